"""CPU tests of the serving entry points' edges: sizes that the host has to get right
before a kernel may run."""
import ctypes

import pytest

P = ctypes.c_void_p
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    from naylis_b200 import _lib, build
    build.build()
    return _lib.load()


def _decode(lib, **kw):
    a = dict(q=P(256), ld=1024, kp=P(256), vp=P(256), pages=4, page=16, table=P(256), tld=4, lens=P(256), max_len=64,
             B=64, H=16, Hk=16, hd=64, scale=0.1, out=P(256), ws=P(256), wsb=1 << 30, stream=None)
    a.update(kw)
    return lib.mom_decode_attn(*a.values())


@pytest.mark.parametrize("B,H,Hk,hd", [(64, 16, 16, 64), (38, 16, 16, 64), (10, 32, 32, 128), (297, 40, 1, 128)])
def test_decode_without_keys_has_its_workspace(lib, B, H, Hk, hd):
    """More lists (sequences x key heads) than CTAs fit the GPU are cut into spans,
    whose cuts are written to the workspace, though no list has a key: a call without
    one is refused."""
    need = lib.mom_decode_attn_workspace_size(B, H, Hk, hd, 0)
    assert need > 0
    none = dict(B=B, H=H, Hk=Hk, hd=hd, ld=H * hd, max_len=0, tld=0, table=None)
    assert _decode(lib, **none, ws=None, wsb=0) == WORKSPACE
    assert _decode(lib, **none, wsb=need - 1) == WORKSPACE
    # few lists: one cluster each, as ever
    assert lib.mom_decode_attn_workspace_size(2, H, Hk, hd, 0) == 0
    assert lib.mom_decode_attn_workspace_size(B, H, Hk, hd, -1) == 0


def test_decode_counts_a_span_in_32_bits(lib):
    """A list's tiles are counted in 32 bits from the start of the one that a span
    begins in, up to the end of the one that it ends in: what does not fit is refused.
    296 CTAs is the least that spans are cut for (head_dim 128)."""
    lists, fits = 1 << 16, (1 << 26) - 256
    long = dict(B=1 << 10, H=64, Hk=64, hd=128, ld=64 * 128, tld=1 << 23, ws=None, wsb=0)
    assert _decode(lib, **long, max_len=fits) == WORKSPACE
    assert _decode(lib, **long, max_len=1 << 26) == INVALID
    assert _decode(lib, **long, max_len=1 << 27) == INVALID
    units = fits // 16 + 6
    assert units + lists * units // 296 + units < 1 << 31


def _prompt(lib, **kw):
    a = dict(q=P(256), qld=128, k=P(256), kld=128, v=P(256), vld=128, Tq=3, Tk=3, H=2, Hk=2, hd=64, scale=0.1,
             plan=P(256), bytes=16 + 152 * 4 + 16 + 16, out=P(256), stream=None)
    a.update(kw)
    return lib.mom_prompt_attn(*a.values())


def test_a_scale_is_positive_and_finite_in_fp32(lib):
    """The kernels take it, times log2 e, in fp32."""
    for scale in (1e-46, 1e-300, 1e39, 1e300, 3e38, 0.0, -1.0, float("inf"), float("nan")):
        assert _prompt(lib, scale=scale) == INVALID, scale
        assert _decode(lib, scale=scale) == INVALID, scale
        assert b"scale" in lib.mom_last_error_string()
    for scale in (1e-44, 1e-30, 2e38):      # on to the next check
        assert _decode(lib, scale=scale, max_len=4096, tld=256, ws=None, wsb=0) == WORKSPACE


def test_tangents_are_noticed():
    import torch
    from torch.autograd import forward_ad

    from naylis_b200 import _lib
    x = torch.ones(3)
    _lib.no_tangent("op", x)
    with forward_ad.dual_level():
        _lib.no_tangent("op", x)
        with pytest.raises(RuntimeError, match="op has no forward-mode"):
            _lib.no_tangent("op", x, forward_ad.make_dual(x, x))


def _logprobs(lib, R, V, back=False):
    if back:
        return lib.mom_logprobs_bwd(P(256), 1, V, P(256), None, P(256), 0, P(256), P(256), P(256), R, V, -100, 1.0, P(256),
                                    None)
    return lib.mom_logprobs_fwd(P(256), 1, V, None, R, V, -100, 1.0, 0, P(256), P(256), None, None, None, None)


def test_logits_rows_are_counted_in_32_bits(lib):
    """The threads' steps past a row's end fit too. (A null pointer stops the calls that
    pass.)"""
    for back in (False, True):
        for V in ((1 << 31) - 1, (1 << 31) - 512, 1 << 31):
            assert _logprobs(lib, 1, V, back) == INVALID and b"geometry" in lib.mom_last_error_string(), V
        assert _logprobs(lib, 1, (1 << 31) - (1 << 17), back) == INVALID
        assert b"null" in lib.mom_last_error_string()
