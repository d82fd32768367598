"""Host-side checks of the cache and window attention operators (no GPU): the C
ABI refuses bad arguments before any CUDA call, the wrappers refuse CPU tensors
and bad options, and the 64-bit restatement agrees with itself.
"""
import ctypes as C

import pytest
import torch

from oracle import kv4_oracle as O


@pytest.fixture(scope="module")
def lib():
    from vc_b200 import _native as N
    from vc_b200 import build as B
    if not N.LIB_PATH.exists():
        B.build()
    return N.load()


def _last(lib):
    return lib.vc_last_error().decode()


P = C.c_void_p(1 << 20)          # never dereferenced: refused first
ST = (4 * 9 * 128, 9 * 128, 128)


def _append(lib, *, dtype=1, B=1, Hq=4, Hkv=2, S=9, D=128, k=P, q=None, qo=None, st=ST, cos=None, sin=None, rows=0,
            rot=0, lengths=P, pool=P, pages=8, page=64, table=P, width=4):
    return lib.vc_kv4_append(k, P, q, qo, dtype, B, Hq, Hkv, S, D, *st, *ST, *ST, *ST, cos, sin, rows, rot, 0, None,
                             lengths, None, pool, pages, page, table, width, None)


@pytest.mark.parametrize("kw,word", [
    ({"dtype": 2}, "dtype"), ({"D": 96}, "head dim"), ({"q": P, "qo": P, "Hq": 3}, "multiple"), ({"B": 0}, "B, Hkv"),
    ({"Hkv": 0, "Hq": 1}, "Hkv"), ({"S": -1}, "S must"), ({"S": 1 << 30}, "S must"), ({"page": 24}, "page_size"),
    ({"page": 512}, "page_size"), ({"pages": 0}, "pages"), ({"width": 1 << 25}, "table_width"),
    ({"table": None}, "page table"), ({"pool": C.c_void_p((1 << 20) + 16)}, "128-byte"), ({"k": None}, "non-null"),
    ({"st": (4 * 9 * 128, 9 * 128, 127)}, "16-byte"), ({"q": P}, "q_out"), ({"rot": 24, "cos": P, "sin": P, "rows": 4}, "rot_dim"),
    ({"rot": 144, "cos": P, "sin": P, "rows": 4}, "rot_dim"), ({"rot": 64, "cos": P, "rows": 4}, "rot_dim"),
    ({"rot": 64, "cos": P, "sin": C.c_void_p((1 << 20) + 4), "rows": 4}, "rot_dim"), ({"lengths": None}, "lengths"),
])
def test_append_refuses(lib, kw, word):
    assert _append(lib, **kw) == 1 and word in _last(lib), _last(lib)


def test_append_of_nothing_is_nothing(lib):
    assert _append(lib, S=0) == 0


def _attend(lib, *, dtype=1, B=1, Hq=4, Hkv=2, Sq=9, D=128, window=0, sinks=0, scale=0.1, most=0, lengths=P, out=P,
            ws=None, wsb=0, page=64, width=4):
    return lib.vc_kv4_attention_fwd(P, dtype, B, Hq, Hkv, Sq, D, *ST, P, 8, page, P, width, lengths, None, 1, window, sinks,
                                    most, scale, out, *ST, ws, wsb, None)


@pytest.mark.parametrize("kw,rc,word", [
    ({"dtype": 2}, 1, "dtype"), ({"Hq": 5}, 1, "multiple"), ({"window": -1}, 1, "window"), ({"sinks": -1}, 1, "sinks"),
    ({"scale": 0.0}, 1, "sm_scale"), ({"scale": float("nan")}, 1, "sm_scale"), ({"lengths": None}, 1, "lengths"),
    ({"out": None}, 1, "out"), ({"most": -1}, 1, "max_length"), ({"Sq": (1 << 30) - 1, "Hq": 8, "Hkv": 1}, 1, "rows"),
    ({"width": 4096}, 4, "workspace"), ({"width": 4096, "ws": C.c_void_p((1 << 20) + 16), "wsb": 1 << 40}, 4, "128-byte"),
])
def test_attention_over_the_cache_refuses(lib, kw, rc, word):
    assert _attend(lib, **kw) == rc and word in _last(lib), _last(lib)


def test_attention_over_the_cache_of_no_queries_is_nothing(lib):
    assert _attend(lib, Sq=0) == 0


def _window(lib, *, dtype=1, Hq=4, Hkv=2, Sq=9, Sk=9, D=128, window=0, scale=0.1, k=P):
    return lib.vc_window_attention_fwd(P, k, P, dtype, 1, Hq, Hkv, Sq, Sk, D, *ST, *ST, *ST, None, 1, window, 0, scale, P,
                                       *ST, None, 0, None)


@pytest.mark.parametrize("kw,rc,word", [
    ({"dtype": 2}, 1, "dtype"), ({"D": 256}, 1, "head dim"), ({"Hkv": 3}, 1, "multiple"), ({"Sk": -1}, 1, "Sk"),
    ({"window": -2}, 1, "window"), ({"scale": -1.0}, 1, "sm_scale"), ({"k": None}, 1, "k must"),
    ({"Sq": 1, "Sk": 1 << 20, "Hq": 2}, 4, "workspace"),
])
def test_window_attention_refuses(lib, kw, rc, word):
    assert _window(lib, **kw) == rc and word in _last(lib), _last(lib)


def test_read_refuses(lib):
    rd = lambda dtype=1, N=4, page=64, start=None: lib.vc_kv4_read(P, 8, page, P, 4, start, 1, 2, N, 128, P, P, dtype, *ST,
                                                                   *ST, None)
    assert rd(dtype=3) == 1 and "dtype" in _last(lib)
    assert rd(N=-1) == 1 and "N must" in _last(lib)
    assert rd(page=8) == 1 and "page_size" in _last(lib)
    assert rd(N=0) == 0


def test_workspace_queries_need_no_device(lib):
    ask = lambda Sq, width, window=0, most=0: lib.vc_kv4_attention_workspace_bytes(1, 28, 4, Sq, 128, 1, window, 0, 64, width, most)
    assert ask(1, 1) == 0                                    # one short sequence: one CTA a head, no partial results
    assert ask(1, 1000) > 0
    assert ask(1, 1000, most=64) == 0                        # the bound counts, not the table
    chunk, bounded = ask(1024, 1000), ask(1024, 1000, window=256)
    assert chunk > 2 * 4 * 64000 * 128 * 2 and 0 < bounded < chunk // 8   # FP16 tiles of what is visible
    assert ask(0, 1000) == 0
    win = lib.vc_window_attention_workspace_bytes
    assert win(1, 8, 8, 4096, 4096, 128, 1, 0, 0) == 0 and win(1, 8, 1, 1, 65536, 128, 1, 0, 0) > 0


def test_wrappers_refuse_cpu_tensors_and_bad_options():
    from vc_b200 import ops
    q, k = torch.zeros((1, 4, 3, 64), dtype=torch.bfloat16), torch.zeros((1, 2, 3, 64), dtype=torch.bfloat16)
    pool, table, n = torch.zeros((4, 2, 4, 1152), dtype=torch.uint8), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    for call in (lambda: ops.kv4_append(pool, table, n, k, k), lambda: ops.kv4_attention(q, pool, table, n),
                 lambda: ops.window_attention(q, k, k), lambda: ops.kv4_read(pool, table, None, 1)):
        with pytest.raises(ValueError, match="no CPU fallback"):
            call()
    with pytest.raises(ValueError, match="tensor_layout"):
        ops.window_attention(q, k, k, tensor_layout="BHSD")
    with pytest.raises(ValueError, match="head_dim"):
        ops.kv4_pool(1, 1, 80)
    with pytest.raises(ValueError, match="page_size"):
        ops.kv4_pool(1, 1, 64, 100)


def test_cache_pages_on_the_host(monkeypatch):
    """Page bookkeeping without a device: allocation, trimming, refusal that changes nothing."""
    from vc_b200 import kv_cache, ops
    calls = []
    monkeypatch.setattr(ops, "kv4_append", lambda pool, table, lengths, k, v, **kw: calls.append(table.clone()))
    c = kv_cache.KV4Cache(2, 1, 64, pages=6, max_tokens=200, page_size=16, window=16, sinks=3, device="cpu")
    k = torch.zeros((2, 1, 40, 64))
    c.append(k, k, counts=[40, 10])
    assert c.free_pages == 6 - 3 - 1 and (calls[0][0, :3] >= 0).all() and calls[0][0, 3] == -1
    assert len(set(calls[0][calls[0] >= 0].tolist())) == 4
    assert c.trim() == 0                       # token 40 sees 25..39: page 1 has 16..31
    c.append(k[:, :, :8], k[:, :, :8], counts=[8, 0])
    assert c.trim() == 1 and c.page_table[0, 1] == -1 and c.page_table[0, 0] >= 0   # 33.. remain visible, sinks stay
    with pytest.raises(RuntimeError, match="pages needed"):
        c.append(k, k, counts=[40, 40])
    assert c.lengths.tolist() == [48, 10]
    c.drop(0)
    assert c.free_pages == 5 and c.lengths.tolist() == [0, 10]


def test_oracle_round_trips_its_own_records():
    g = torch.Generator().manual_seed(3)
    x = torch.randn((2, 5, 128), generator=g) * 3
    u, s, m = O.quantise(x)
    y = O.dequantise(u, s, m)
    assert u.min() == 0 and u.max() == 15
    step = s.repeat_interleave(64, -1)
    assert ((x - y).abs() <= step * 0.5 + m.abs().repeat_interleave(64, -1) * 2.0 ** -8 + step * 2.0 ** -4).all()
    pool = torch.zeros((1, 1, 1, 18 * 128), dtype=torch.uint8)
    rec = pool[0, 0, 0]
    for t in range(5):
        rec[t * 64:(t + 1) * 64] = (u[0, t, 0::2].int() | (u[0, t, 1::2].int() << 4)).to(torch.uint8)
        rec[2048 + t * 8:2048 + t * 8 + 8] = torch.stack((s[0, t], m[0, t]), -1).to(torch.bfloat16).view(torch.uint8).flatten()
    k, _ = O.decode(pool, torch.zeros(1, dtype=torch.int32), 0, 5)
    assert torch.equal(k, y[0])


def test_direct_calls_leave_what_they_do_not_take_to_the_wrappers():
    from vc_b200 import _native as N
    from vc_b200 import build as B
    if not N.CALLS_PATH.exists():
        B.build()
    f = N.calls()
    x = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16)
    pool, table, n = torch.zeros((2, 2, 1, 1152), dtype=torch.uint8), torch.zeros((1, 2), dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    assert f.kv4_append(pool, table, n, x, x, None, None, None, None, None, False, "HND") is NotImplemented
    assert f.kv4_read(pool, table, n, 1, torch.float16, "HND") is NotImplemented
    assert f.kv4_attention(x, pool, table, n, None, True, None, 0, None, None, "HND") is NotImplemented
    assert f.window_attention(x, x, x, None, 0, True, None, None, "HND") is NotImplemented
    for name in ("kv4_append", "kv4_read", "kv4_attention", "window_attention"):
        assert getattr(f, name)() is NotImplemented and getattr(f, name)(1, "a", None) is NotImplemented
    with pytest.raises(TypeError):
        f.bind(1)
