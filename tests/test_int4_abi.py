"""CPU tests of the 4-bit cache's and the drafts' entry points of the C ABI: the arguments
they reject before any device work, and the sizes that the host has to get right."""
import ctypes
import os
import re

import pytest

P = ctypes.c_void_p
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    from naylis_b200 import _lib, build
    build.build()
    return _lib.load()


def _rope(lib, **kw):
    a = dict(qkv=P(256), ld=384, cos=P(256), sin=P(256), n_pos=8, pos=P(256), pt=3, slots=P(256), st=3, T=2, H=2, Hk=2,
             hd=64, pages=4, page=16, kp=P(256), vp=P(256), sc=P(256), q=P(256), k=None, v=None, stream=None)
    a.update(kw)
    return lib.mom_rope_append_int4(*a.values())


def _decode(lib, **kw):
    a = dict(q=P(256), ld=128, kp=P(256), vp=P(256), sc=P(256), pages=4, page=16, table=P(256), tld=4, lens=P(256),
             new=None, max_len=64, B=2, n=1, H=2, Hk=2, hd=64, scale=0.1, out=P(256), ws=P(256), wsb=1 << 30, stream=None)
    a.update(kw)
    return lib.mom_decode_attn_int4(*a.values())


def _verify(lib, **kw):
    a = dict(x=P(256), dt=1, ls=60, lr=20, q=P(256), qs=40, qr=20, d=P(256), u=P(256), n=None, B=3, K=2, V=20, T=1.0,
             tok=P(256), acc=P(256), stream=None)
    a.update(kw)
    return lib.mom_verify_drafts(*a.values())


def test_append_refuses(lib):
    for kw in (dict(H=3), dict(Hk=0), dict(ld=383), dict(ld=376), dict(page=12), dict(page=4), dict(page=512), dict(T=-1),
               dict(pt=0), dict(st=1), dict(qkv=P(264)), dict(qkv=None), dict(kp=None), dict(sc=None), dict(q=None),
               dict(n_pos=-1), dict(sc=P(264)), dict(k=P(260)), dict(v=P(8)), dict(pages=-1)):
        assert _rope(lib, **kw) == INVALID, kw
    assert _rope(lib, hd=96) == UNSUPPORTED
    assert _rope(lib, T=0, qkv=None) == OK
    # the cache's rows are counted in 32 bits
    assert _rope(lib, pages=(1 << 26) + 1) == INVALID and b"2^31" in lib.mom_last_error_string()


def test_decode_refuses(lib):
    for kw in (dict(H=3), dict(B=-1), dict(B=70000), dict(n=0), dict(n=65), dict(max_len=65), dict(max_len=-1),
               dict(ld=120), dict(ld=132), dict(scale=float("nan")), dict(scale=0.0), dict(scale=1e-46), dict(q=None),
               dict(lens=None), dict(table=None), dict(kp=None), dict(sc=None), dict(out=P(260)), dict(page=20),
               dict(sc=P(264)), dict(pages=(1 << 26) + 1)):
        assert _decode(lib, **kw) == INVALID, kw
    assert _decode(lib, hd=32) == UNSUPPORTED
    assert _decode(lib, B=0, q=None) == OK


@pytest.mark.parametrize("B,n,H,Hk,hd", [(2, 1, 2, 2, 64), (38, 1, 16, 16, 64), (9, 5, 32, 4, 128), (70, 64, 40, 1, 64)])
@pytest.mark.parametrize("max_len", [0, 64, 1 << 20])
def test_decode_takes_its_workspace(lib, B, n, H, Hk, hd, max_len):
    """Lists without keys write their cuts too: a call without the workspace is refused."""
    need = lib.mom_decode_attn_int4_workspace_size(B, n, H, Hk, hd, max_len)
    call = dict(B=B, n=n, H=H, Hk=Hk, hd=hd, ld=H * hd, max_len=max_len, tld=max_len // 16)
    if need:
        assert _decode(lib, **call, ws=None, wsb=0) == WORKSPACE
        assert _decode(lib, **call, wsb=need - 1) == WORKSPACE
    else:
        lists = B * Hk * -(-(n * H // Hk) // 8)
        assert lists <= 148 * 4 and max_len < 1 << 20
    assert lib.mom_decode_attn_int4_workspace_size(B, n, H, Hk, hd, -1) == 0
    assert lib.mom_decode_attn_int4_workspace_size(B, 0, H, Hk, hd, 64) == 0


def test_decode_counts_a_span_in_32_bits(lib):
    many = dict(B=1 << 10, n=1, H=64, Hk=64, hd=128, ld=64 * 128, tld=1 << 23, ws=None, wsb=0)
    assert _decode(lib, **many, max_len=(1 << 26) - 256) == WORKSPACE
    assert _decode(lib, **many, max_len=1 << 26) == INVALID
    lists, units = 1 << 16, (1 << 26) // 32 + 6
    assert units + lists * units // 444 + units < 1 << 31
    assert _decode(lib, B=65535, n=64, H=512, Hk=2, ld=512 * 64) == INVALID      # 2^30 rows


def test_verify_refuses(lib):
    for kw in (dict(dt=2), dict(B=-1), dict(B=70000), dict(K=-1), dict(K=33), dict(V=0), dict(V=1 << 31),
               dict(V=(1 << 31) - 1024), dict(T=-1.0), dict(T=float("nan")), dict(T=1e-7), dict(T=1e7), dict(x=None),
               dict(d=None), dict(u=None), dict(tok=None), dict(acc=None), dict(x=P(257)), dict(q=P(257)), dict(lr=-1),
               dict(qs=-1)):
        assert _verify(lib, **kw) == INVALID, kw
    assert _verify(lib, B=0, x=None) == OK


def test_the_python_calls_refuse_what_is_not_on_a_gpu():
    import torch

    from naylis_b200 import attention, scoring
    k = torch.zeros(2, 1, 16, 32, dtype=torch.uint8)
    s = torch.zeros(2, 1, 16, 1, 4, dtype=torch.bfloat16)
    q = torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16)
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="decode_attention_int4"):
        attention.decode_attention_int4(q, k, k, s, i[None], i)
    with pytest.raises(RuntimeError, match="rope_append_int4"):
        attention.rope_append_int4(q.view(1, 64), s, s, i, k, k, s, i, n_heads=1)
    with pytest.raises(RuntimeError, match="verify_drafts"):
        scoring.verify_drafts(torch.zeros(1, 2, 5), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))


def test_packed_calls(lib):
    """Entries of call_on()'s short way are the header's, and take all of their arguments."""
    from naylis_b200 import _lib
    header = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "naylis_mom.h")).read()
    entries = {f"mom_{n.lower()}": int(i) for n, i in re.findall(r"MOM_CALL_(\w+) = (\d+)", header)}
    assert entries == {name: i for name, (i, _, _) in _lib._PACKED.items()}
    for name, (entry, pack, n) in _lib._PACKED.items():
        kinds = _lib.SIGNATURES[name][1]
        args = pack(*(0.5 if k is ctypes.c_double else 0 for k in kinds))
        assert len(args) == 8 * n == 8 * len(kinds)
        one = getattr(lib, name)(*(0.5 if k is ctypes.c_double else 0 for k in kinds))
        error = _lib.last_error()
        packed = lib.mom_call_packed(entry, args, n)
        assert packed == one and one != 0 and _lib.last_error() == error
        assert lib.mom_call_packed(entry, args, n - 1) == 1 and "packed arguments" in _lib.last_error()
    assert lib.mom_call_packed(len(entries), b"", 0) == 1 and "no packed entry" in _lib.last_error()
