"""CPU tests of the serving and scoring entry points of the C ABI: the prompt plan
(host code) and the arguments they reject before any device work."""
import ctypes

import numpy as np
import pytest

P = ctypes.c_void_p
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    from naylis_b200 import _lib, build
    build.build()
    return _lib.load()


def _plan(lib, ql, kl=None, H=4, Hk=4):
    q = np.asarray(ql, dtype=np.int64)
    k = None if kl is None else np.asarray(kl, dtype=np.int64)
    size = lib.mom_prompt_plan_size(q.ctypes.data, len(ql), H, Hk)
    buf = np.full(size, 0xAB, dtype=np.uint8)
    rc = lib.mom_prompt_plan(q.ctypes.data, None if k is None else k.ctypes.data, len(ql), H, Hk, buf.ctypes.data, size)
    assert rc == OK
    n = sum(-(-x // 256) for x in ql)
    words = buf.view(np.int32)
    assert not words[:4].any()
    tiles = words[4:4 + 4 * n].reshape(n, 4)
    first = words[4 + 4 * n:][:149]
    items = words[4 + 4 * n + 152:].reshape(-1, 2)
    assert len(items) == n * H
    return tiles, first, items


@pytest.mark.parametrize("ql,kl", [([1], None), ([256, 257, 0, 1, 1000], None), ([5, 300], [400, 10]), ([0, 0], None)])
@pytest.mark.parametrize("H,Hk", [(4, 4), (4, 2), (6, 2)])
def test_plan_covers_every_row_and_head_once(lib, ql, kl, H, Hk):
    tiles, first, items = _plan(lib, ql, kl, H, Hk)
    seen = np.zeros((sum(ql), H), dtype=int)
    q0 = np.concatenate([[0], np.cumsum(ql)])
    k0 = np.concatenate([[0], np.cumsum(kl or ql)])
    for a, rows, k, vis in tiles:
        assert 1 <= rows <= 256
        i = int(np.searchsorted(q0, a, side="right") - 1)
        assert a + rows <= q0[i + 1] and k == k0[i]
        assert vis == (kl or ql)[i] - ql[i] + (a - q0[i]) + 1
    assert first[0] == 0 and (np.diff(first) >= 0).all()
    for t, rem in items[:first[148]]:
        a, rows = tiles[t][:2]
        if H // Hk % 2:                      # a head, all rows
            seen[a:a + rows, rem] += 1
        else:                                # two heads, rows 0 .. 127 or 128 .. 255
            sub, pair = (1, rem) if rem < H // 2 else (0, rem - H // 2)
            assert rows > 128 * sub
            seen[a + 128 * sub:a + min(rows, 128 * sub + 128), 2 * pair:2 * pair + 2] += 1
    assert (seen == 1).all()


def test_plan_levels_the_work(lib):
    """Longest first to the least busy: nobody is above the mean by more than the
    largest item."""
    rng = np.random.RandomState(0)
    ql = [int(x) for x in np.exp(rng.uniform(0, np.log(4000), 40))]
    tiles, first, items = _plan(lib, ql, None, 8, 8)
    cost = (tiles[:, 3] + tiles[:, 1] - 1 + 127) // 128 + 1.5
    per = [cost[items[first[c]:first[c + 1], 0]] for c in range(148)]
    load = np.array([x.sum() for x in per])
    assert load.max() <= load.mean() + cost.max()
    assert all((np.diff(x) <= 0).all() for x in per)


def test_plan_refuses(lib):
    one = np.asarray([-1], dtype=np.int64)
    assert lib.mom_prompt_plan_size(one.ctypes.data, 1, 4, 4) == 0 and b"lengths" in lib.mom_last_error_string()
    big = np.asarray([1 << 30, 1 << 30], dtype=np.int64)
    assert lib.mom_prompt_plan_size(big.ctypes.data, 2, 4, 4) == 0
    two = np.asarray([300, 4], dtype=np.int64)
    assert lib.mom_prompt_plan_size(two.ctypes.data, 2, 4, 3) == 0
    buf = np.zeros(4096, dtype=np.uint8)
    assert lib.mom_prompt_plan(two.ctypes.data, None, 2, 4, 4, buf.ctypes.data, 32) == WORKSPACE
    assert lib.mom_prompt_plan(two.ctypes.data, None, 2, 4, 4, None, 4096) == INVALID
    assert lib.mom_prompt_plan(two.ctypes.data, None, 2, 0, 4, buf.ctypes.data, 4096) == INVALID


def _rope(lib, **kw):
    a = dict(qkv=P(256), ld=384, cos=P(256), sin=P(256), n_pos=8, pos=P(256), pt=3, slots=P(256), st=3, T=2, H=2, Hk=2,
             hd=64, pages=4, page=16, kp=P(256), vp=P(256), q=P(256), k=None, stream=None)
    a.update(kw)
    return lib.mom_rope_append(*a.values())


def _decode(lib, **kw):
    a = dict(q=P(256), ld=128, kp=P(256), vp=P(256), pages=4, page=16, table=P(256), tld=4, lens=P(256), max_len=64,
             B=2, H=2, Hk=2, hd=64, scale=0.1, out=P(256), ws=P(256), wsb=1 << 30, stream=None)
    a.update(kw)
    return lib.mom_decode_attn(*a.values())


def _prompt(lib, **kw):
    a = dict(q=P(256), qld=128, k=P(256), kld=128, v=P(256), vld=128, Tq=3, Tk=3, H=2, Hk=2, hd=64, scale=0.1,
             plan=P(256), bytes=16 + 152 * 4 + 32, out=P(256), stream=None)
    a.update(kw)
    return lib.mom_prompt_attn(*a.values())


def _lp(lib, **kw):
    a = dict(x=P(256), dt=1, ld=20, t=P(256), R=2, V=20, ignore=-100, T=1.0, top=2, lp=P(256), ent=P(256), tl=P(256),
             ti=P(256), stats=P(256), stream=None)
    a.update(kw)
    return lib.mom_logprobs_fwd(*a.values())


def _lpb(lib, **kw):
    a = dict(x=P(256), dt=1, ld=20, t=P(256), stats=P(256), ti=P(256), top=2, g=P(256), h=P(256), a=P(256), R=2, V=20,
             ignore=-100, T=1.0, dx=P(256), stream=None)
    a.update(kw)
    return lib.mom_logprobs_bwd(*a.values())


def test_bad_arguments_fail_before_device_work(lib):
    for kw in (dict(H=3), dict(Hk=0), dict(ld=383), dict(ld=376), dict(page=12), dict(page=4), dict(page=512), dict(T=-1),
               dict(pt=0), dict(st=1), dict(qkv=P(264)), dict(qkv=None), dict(kp=None), dict(q=None), dict(n_pos=-1)):
        assert _rope(lib, **kw) == INVALID, kw
    assert _rope(lib, hd=96) == UNSUPPORTED
    assert _rope(lib, T=0, qkv=None) == OK
    for kw in (dict(H=3), dict(B=-1), dict(B=70000), dict(max_len=65), dict(max_len=-1), dict(ld=120), dict(ld=132),
               dict(scale=float("nan")), dict(q=None), dict(lens=None), dict(table=None), dict(out=P(260)), dict(page=20)):
        assert _decode(lib, **kw) == INVALID, kw
    assert _decode(lib, hd=32) == UNSUPPORTED
    assert _decode(lib, B=0, q=None) == OK
    long = dict(tld=1 << 16, max_len=1 << 20)
    need = lib.mom_decode_attn_workspace_size(2, 2, 2, 64, 1 << 20)
    assert need > 0 and _decode(lib, **long, ws=None, wsb=0) == WORKSPACE
    assert _decode(lib, **long, wsb=need - 1) == WORKSPACE
    for kw in (dict(H=3), dict(Tq=-1), dict(kld=64), dict(vld=132), dict(scale=float("inf")), dict(plan=None),
               dict(bytes=16), dict(bytes=40), dict(q=P(264)), dict(out=None), dict(v=None)):
        assert _prompt(lib, **kw) == INVALID, kw
    assert _prompt(lib, hd=256) == UNSUPPORTED
    assert _prompt(lib, Tq=0, q=None) == OK
    for kw in (dict(dt=2), dict(ld=19), dict(V=0), dict(R=-1), dict(T=0.0), dict(T=float("nan")), dict(T=1e-60),
               dict(top=33), dict(top=21), dict(top=-1), dict(x=None), dict(t=None), dict(ti=None), dict(x=P(257)),
               dict(stats=P(264))):
        assert _lp(lib, **kw) == INVALID, kw
    assert _lp(lib, R=0, x=None) == OK
    for kw in (dict(stats=None), dict(dx=None), dict(ti=None), dict(dx=P(257)), dict(T=-1.0)):
        assert _lpb(lib, **kw) == INVALID, kw


def test_decode_refuses_more_keys_than_it_counts(lib):
    many = dict(B=65535, H=64, Hk=64, ld=4096, tld=1 << 20, max_len=1 << 24)
    assert _decode(lib, **many) == INVALID
    assert lib.mom_decode_attn_workspace_size(65535, 64, 64, 64, 1 << 20) > 0
    assert lib.mom_decode_attn_workspace_size(2, 2, 2, 64, 0) == 0      # few short lists need none
