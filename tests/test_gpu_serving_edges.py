"""GPU tests of the serving operators at their edges: calls without keys, values that
are not finite, scales and lengths at the ends of their ranges."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _rand(seed, *shape, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * scale).to(torch.bfloat16).to(DEV)


@pytest.mark.parametrize("B,H,Hk,hd", [(64, 16, 16, 64), (40, 32, 32, 128), (300, 40, 1, 128), (2, 4, 2, 64)])
@pytest.mark.parametrize("pages", [0, 3])
def test_decode_without_keys(B, H, Hk, hd, pages):
    """max_len 0: zeros for sequences without keys, NaN for those that claim some, as
    many lists as there are."""
    from naylis_b200 import attention
    q = _rand(1, B, H, hd)
    kp, vp = _rand(2, 3, Hk, 16, hd), _rand(3, 3, Hk, 16, hd)
    table = torch.zeros(B, pages, dtype=torch.int32, device=DEV)
    lens = torch.zeros(B, dtype=torch.int32, device=DEV)
    lens[B // 2] = -4
    assert bool((attention.decode_attention(q, kp, vp, table, lens, max_len=0) == 0).all())
    lens[0], lens[B - 1] = 1, 1 << 30
    out = attention.decode_attention(q, kp, vp, table, lens, max_len=0)
    assert bool(torch.isnan(out[[0, B - 1]]).all()) and bool((out[1:B - 1] == 0).all())
