"""GPU test of the one rounding in which rope_append_int4's scale could be taken two ways."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
def test_the_scale_is_a_product(hd):
    """scale = bf16((greatest - least) * fp32(1 / 15)): fp32's 1 / 15 is above 1 / 15, so that a range whose
    fifteenth is a tie of bf16's (1.25 and 1.2578125 here) goes up, where the quotient goes to the even 1.25."""
    from naylis_b200 import attention
    least, most = -0.05859375, 18.75
    span = torch.tensor(most) - torch.tensor(least)
    assert float((span / 15).to(torch.bfloat16)) == 1.25 and float((span * (1.0 / 15)).to(torch.bfloat16)) == 1.2578125
    k = torch.zeros(1, 1, 16, hd // 2, dtype=torch.uint8, device="cuda")
    v, scales = torch.zeros_like(k), torch.zeros(1, 1, 16, hd // 64, 4, dtype=torch.bfloat16, device="cuda")
    qkv = torch.zeros(1, 3 * hd, dtype=torch.bfloat16, device="cuda")
    qkv[:, 0::64], qkv[:, 1::64] = least, most
    cos, sin = torch.ones(1, hd, device="cuda"), torch.zeros(1, hd, device="cuda")
    at = torch.zeros(1, dtype=torch.int64, device="cuda")
    _, got_k, got_v = attention.rope_append_int4(qkv, cos, sin, at, k, v, scales, at, n_heads=1, want_kv=True)
    row = scales[0, 0, 0].float().cpu()
    assert torch.equal(row[:, 0::2], torch.full((hd // 64, 2), 1.2578125))
    assert torch.equal(row[:, 1::2], torch.full((hd // 64, 2), least))
    stands = (torch.tensor(1.2578125) * 15 + least).to(torch.bfloat16)      # number 15
    assert bool((got_k[0, 0, 1::64].cpu() == stands).all()) and bool((got_v[0, 0, 1::64].cpu() == stands).all())
