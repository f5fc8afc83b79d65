"""GPU parity: attention over a shared prefix where values or scores are not of ordinary size.

Bound of the first tests, of the error's norm over all outputs, derived from what the kernel rounds.  A probability
times its V scale is rounded to fp16, half a step of which is 2^-11 of it: an error of variance
at most (2^-11 p v)^2 / 3 for every token, and of either sign.  The output is rounded to its type:
half a step is 2^-11 of it (2^-25 at least) or 2^-8 (bf16), of variance a third of the
square.  Their sum over tokens and outputs is the square of the norm that is expected at most; what
is left (fp32 sums, exp2) is below a tenth of it, and the norm of 10^4 errors and more is within
a tenth of what is expected.  No term of the bound is absolute in V: V ten thousand times smaller
has to come out as precisely."""
import math

import pytest
import torch

from test_gpu_shared_attn import BF16, DEV, F16, Case

pytestmark = pytest.mark.gpu
PART, V_SCALES = 2208, 2112     # bytes of a kv head's part of a record, and where its V scales lie


def _scale_values(c, factor):
    """c with every V times factor(number of the token in its sequence), a power of two: exact in the
    records' V scales; zones (their V rounded to fp16) take that of the last INT4 token."""
    part = c.pool.data.view(-1, c.hkv, PART)
    done = set()
    for b in range(c.B):
        n = c.shared + c.own[b]
        f = torch.tensor([factor(t) for t in range(n)], dtype=torch.float64, device=DEV)
        zone = factor(max(n - 1, 0))
        for lo in range(0, n, 16):
            i = int(c.bt[b, lo // 16])
            if i not in done:
                done.add(i)
                s = part[i, :, V_SCALES:V_SCALES + 64].contiguous().view(torch.float32)
                s[:, :min(16, n - lo)] *= f[lo:lo + 16].float()
                part[i, :, V_SCALES:V_SCALES + 64] = s.view(torch.uint8)
        at, values = 0, []
        for x in c.values[b]:
            k = x.shape[1]
            values.append(x * f[at:at + k, None] if at < n else (x.half() * zone).double())
            at += k
        c.values[b] = values
    for z, _, _ in c.zones:
        z.v.mul_(factor(c.max_len - 1))
    return c


def _check(c, out_dtype, **kw):
    out = c.run(out_dtype=out_dtype, **kw)
    torch.cuda.synchronize()
    c.pool.check_errors()
    rep, off, bound = c.hq // c.hkv, 0.0, 0.0
    for b in range(c.B):
        k, v = torch.cat(c.keys[b], 1), torch.cat(c.values[b], 1)
        q = c.q[b].double().view(c.hkv, rep, 128)
        for h in range(c.hkv):
            p = torch.softmax(q[h] @ k[h].t() / math.sqrt(128), -1)
            want = p @ v[h]
            got = out[b, h * rep:(h + 1) * rep].double()
            assert bool(torch.isfinite(got).all())
            half = want.abs() * 2.0 ** -8 if out_dtype == BF16 else (want.abs() * 2.0 ** -11).clamp(min=2.0 ** -25)
            off += float(((got - want) ** 2).sum())
            bound += float(((2.0 ** -22 * (p * p) @ (v[h] * v[h]) + half ** 2) / 3).sum())
    print("  error norm %.3e, %.2f of what is expected" % (off ** 0.5, (off / bound) ** 0.5), flush=True)
    assert off <= 1.2 ** 2 * bound


@pytest.mark.parametrize("power,out_dtype", [(0, F16), (-6, F16), (-8, F16), (-10, F16), (-12, BF16), (-16, BF16), (-20, BF16),
                                             (-40, BF16), (4, F16), (8, F16), (12, F16), (12, BF16), (30, BF16)])
def test_values_of_any_size(power, out_dtype):
    print("case: V x 2^%d, output %s" % (power, out_dtype), flush=True)
    zone = 30 if -12 <= power <= 8 else 0      # (fp16 holds no smaller or larger ones)
    c = Case(40, 1, 4, 32, 8, 16384, [300, 40, 0, 1000], zone and 16, [zone, zone, zone // 2, 0])
    _check(_scale_values(c, lambda t: 2.0 ** power), out_dtype)


@pytest.mark.parametrize("r,hq,hkv", [(3, 8, 8), (9, 32, 8), (13, 28, 4), (20, 24, 8)])
@pytest.mark.parametrize("name", ["small ones first", "large ones first", "in turn", "one large block"])
def test_values_of_many_sizes(name, r, hq, hkv):
    print("case: %s, %d x %d/%d" % (name, r, hq, hkv), flush=True)
    factor = {"small ones first": lambda t: 2.0 ** (t // 64 % 60 - 50), "large ones first": lambda t: 2.0 ** (10 - t // 64 % 24),
              "in turn": lambda t: 2.0 ** (t // 16 * 5 % 17 - 9), "one large block": lambda t: 2.0 ** (9 if t // 16 == 71 else -7)}[name]
    c = Case(41, 1, r, hq, hkv, 3200, [(70 * i) % 301 for i in range(r)])
    _check(_scale_values(c, factor), BF16)


def test_small_values_beside_decode_attention():
    """No less precise than the same tokens' decode_attention, whose reference is the maximum itself."""
    from heterokv import ops
    for power in (0, -3, -6, -8, -10):
        c = _scale_values(Case(42, 1, 2, 32, 8, 16384, [300, 20]), lambda t: 2.0 ** power)
        a, b = c.run(), ops.decode_attention(c.q, pool=c.pool, block_table=c.bt, int4_lens=c.lens, int4_max_len=c.max_len)
        want, _ = c.exact()
        ea, eb = float((a.double() - want).norm()), float((b.double() - want).norm())
        print("  V x 2^%d: error norm %.3e, decode_attention %.3e" % (power, ea, eb), flush=True)
        assert ea <= 1.1 * eb      # (equal where both are rounded alike: 8192 errors, within a tenth)


def test_scores_of_minus_infinity_before_small_ones():
    """Keys that hold -inf take their tokens out (all queries are positive there): three tiles of 16 in
    four.  The others' scores are some 120 below 0 in the log2 domain, which softmax does not see."""
    print("case: 40 x 32/8, 512 fp16 tokens, 384 of them at -inf", flush=True)
    c = Case(50, 1, 40, 32, 8, 0, 0, 0, [512] * 40)
    z, _, n = c.zones[0]
    g = torch.Generator(device=DEV).manual_seed(51)
    k = torch.randn((40, 8, n, 128), generator=g, device=DEV).half()
    v = torch.randn((40, 8, n, 128), generator=g, device=DEV).half()
    out = torch.arange(n, device=DEV) // 16 % 4 != 3
    k[:, :, out, 0] = float("-inf")
    k[..., 1] = -941.0
    c.q[..., 0], c.q[..., 1] = c.q[..., 0].abs() + 0.01, 1.0
    z.write(k, v, 0)
    c.keys = [[k[b][:, ~out].double()] for b in range(40)]
    c.values = [[v[b][:, ~out].double()] for b in range(40)]
    c.check(int4_max_len=0, pool=None, block_table=None, int4_lens=None)


@pytest.mark.parametrize("shared", [512, 1024, 1600, 2048, 3328, 4000, 6000, 9600])
def test_what_the_workspace_held_before_does_not_matter(shared):
    """Of sequences that do not hold the prefix, its states are not written: NaN stays there."""
    c = Case(52, 1, 3, 32, 8, shared, [20, 3, 0])
    ws = torch.full((32 << 20,), 255, dtype=torch.uint8, device=DEV)
    for keep in ([7, shared - 1, 16], [shared + 20, 5, 0], [0, 0, 1], [1, shared + 3, shared]):
        ws.fill_(255)
        c.check(keep=keep, int4_lens=torch.tensor(keep, dtype=torch.int32, device=DEV), workspace=ws)
