"""GPU parity: attention over a shared prefix where scores or values are not of ordinary size."""
import pytest
import torch

from test_gpu_shared_attn import DEV, F16, Case

pytestmark = pytest.mark.gpu


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
