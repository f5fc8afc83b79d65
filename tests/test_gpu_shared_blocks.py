"""GPU: every block of a long prefix counts once.  All keys are equal, so that every token weighs
1 / T, and V is not zero in one block alone: a lost block gives 0, a doubled one twice the output.

Bound, relative: P (equal to the maximum) is rounded to fp16 by 2^-11 of itself at most, its sum is
not, and the output by 2^-8 (bf16); codes and fp32 sums of T equal terms (T 2^-24 at most) add less."""
import pytest
import torch

from test_gpu_shared_attn import DEV

pytestmark = pytest.mark.gpu
EACH = 2.0 ** -8 + 2.0 ** -11


def _borders(blocks, seed):
    """Blocks at the borders of id windows (64), of 8 waves' runs and of ranges, the first and the last
    ones, and others."""
    at = {0, 1, 2, blocks - 1, blocks - 2, blocks - 3}
    for step in (64, 128, 512, 1024):
        for x in range(step, blocks, step * max(1, blocks // step // 4)):
            at |= {x - 1, x, x + 1}
    for parts in (2, 3, 5, 8, 16, 24, 32, 40, 64, 256):
        for k in range(1, parts, max(1, parts // 6)):
            x = blocks * k // parts
            at |= {x - 1, x, x + 1, x + 2}
    g = torch.Generator().manual_seed(seed)
    at |= set(torch.randint(0, blocks, (24,), generator=g).tolist())
    return sorted(x for x in at if 0 <= x < blocks)


@pytest.mark.parametrize("r,hq,hkv,shared,own", [(2, 32, 8, 1024, 40), (1, 4, 4, 40000, 0), (2, 8, 4, 126912, 40),
                                                 (8, 28, 4, 28624, 200), (5, 32, 8, 4112, 9000), (20, 16, 4, 16400, 33),
                                                 (3, 8, 8, 80016, 20), (70, 2, 2, 2064, 48)])
def test_every_block_counts_once(r, hq, hkv, shared, own):
    from heterokv import ops
    print("case: %d x %d/%d, %d shared, %d own" % (r, hq, hkv, shared, own), flush=True)
    n, mine = shared // 16, -(-own // 16)
    total = n + r * mine
    pool = ops.Int4Pool(total, hkv, DEV)
    g = torch.Generator(device=DEV).manual_seed(shared)
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    bt = torch.cat([perm[:n].expand(r, n), perm[n:].view(r, mine)], 1).contiguous()
    k = torch.randn((1, hkv, 1, 128), generator=g, device=DEV).half()
    zero = torch.zeros((1, hkv, 16, 128), device=DEV).half()
    every = torch.arange(total, dtype=torch.int32, device=DEV)[None]
    ops.pack_tokens(pool, k.expand(1, hkv, 16 * total, 128), torch.zeros((1, hkv, 16 * total, 128), device=DEV).half(), 0, every)
    # 16 different tokens, whose codes are exact: 0 .. 15 in turn
    v = ((torch.arange(128, device=DEV)[None] + torch.arange(16, device=DEV)[:, None]) % 16).half().expand(1, hkv, 16, 128).contiguous()
    kk = k.expand(1, hkv, 16, 128).contiguous()
    q = torch.randn((r, hq, 128), generator=g, device=DEV).half()
    lens = torch.tensor([shared + own - (i * 3) % (own + 1) for i in range(r)], dtype=torch.int32, device=DEV)
    part = v[0, 0].double().sum(0)

    def check(block, sequences, lens=lens):
        ids = bt[sequences[0], block:block + 1][None]
        ops.pack_tokens(pool, kk, v, 0, ids)
        out = ops.shared_prefix_attention(q, n, pool=pool, block_table=bt, int4_lens=lens, int4_max_len=shared + own,
                                          out_dtype=torch.bfloat16)
        held = [max(0, min(16, int(x) - 16 * block)) for x in lens.tolist()]
        for b in range(r):
            want = v[0, 0, :held[b]].double().sum(0) / max(int(lens[b]), 1) if b in sequences else torch.zeros_like(part)
            got = out[b].double()
            assert bool(((got - want).abs() <= EACH * want.abs()).all()), (block, b)
        ops.pack_tokens(pool, kk, zero, 0, ids)

    for block in _borders(n, shared):
        check(block, list(range(r)))
    for b in sorted({0, r - 1}):
        for block in sorted({0, 1, mine // 2, mine - 2, mine - 1} & set(range(mine))):
            check(n + block, [b])
    # a sequence that is a token short of the prefix has all of its blocks
    short = lens.clone()
    short[r - 1] = shared - 1
    for block in _borders(n, shared + 1)[::3] + [n - 1]:
        check(block, list(range(r)), short)
    pool.check_errors()
