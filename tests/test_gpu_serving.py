"""The paged 4-bit cache and window attention on the GPU, against their 64-bit
restatement (oracle/kv4_oracle.py).

Cache contents and rotated queries are compared exactly (the definition fixes
every FP32 rounding); attention within the bound that the oracle derives per
element from the data (``attention_tolerance``), for operands of 8 significant
bits (BF16 probabilities) or 11 (FP16).  Every test ends with a clean device
error word.
"""
import math

import pytest
import torch

from oracle import kv4_oracle as O

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def ops(cuda_device):
    from vc_b200 import ops as o
    o.error_word(0, clear=True)
    return o


@pytest.fixture(autouse=True)
def clean_error_word(ops):
    yield
    assert ops.error_word(0, clear=True) == 0


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, dtype=BF):
    return torch.randn(shape, generator=g).to(dtype)


def _table(g, B, per, spare=2):
    """Scattered pages; one entry more than needed a row, invalid."""
    t = torch.randperm(B * per + spare, generator=g)[: B * per].to(torch.int32).view(B, per)
    return torch.cat((t, torch.full((B, 1), -1, dtype=torch.int32)), 1).contiguous(), B * per + spare


def _garbage_pool(g, pages, H, page, D):
    """Pages whose every byte is an earlier user's: NaN and infinite scales among them."""
    pool = torch.randint(0, 256, (pages, H, page // 16, 18 * D), generator=g, dtype=torch.uint8)
    pool[..., 16 * D::4] = 0xC0
    pool[..., 16 * D + 1::4] = 0x7F   # half of the scales NaN
    return pool


def _filled(ops, g, B, H, D, page, lengths, spread=1.0, dtype=BF):
    """A cache with K/V of ``lengths`` tokens written by kv4_append, between garbage."""
    most = max(1, max(lengths))
    table, pages = _table(g, B, -(-most // page))
    pool = _garbage_pool(g, pages, H, page, D).cuda()
    k, v = (_randn(g, B, H, most, D, dtype=dtype) * spread for _ in range(2))
    k = k + torch.randn((1, H, 1, D), generator=g).to(dtype)
    n = torch.tensor(lengths, dtype=torch.int32)
    zero = torch.zeros(B, dtype=torch.int32, device="cuda")
    ops.kv4_append(pool, table.cuda(), zero, k.cuda(), v.cuda(), counts=n.cuda())
    return pool, table, n


# ---------------------------------------------------------------------------
# append and read
# ---------------------------------------------------------------------------
APPEND = [  # B, S, Hq, Hkv, D, page, dtype, layout, R, interleaved, past
    (1, 1, 2, 1, 128, 64, BF, "HND", 128, False, 0),
    (3, 1, 7, 1, 64, 16, HF, "NHD", 64, True, 15),
    (2, 37, 6, 3, 128, 16, BF, "NHD", 64, False, 16),
    (2, 130, 8, 2, 128, 128, HF, "HND", 96, True, 127),
    (1, 70, 5, 5, 64, 32, BF, "HND", 32, False, 1),
    (2, 17, 4, 4, 64, 256, HF, "NHD", 16, False, 300),
    (1, 5, 3, 1, 128, 64, BF, "HND", 0, False, 62),
    (5, 300, 2, 2, 128, 64, BF, "NHD", 128, False, 33),
]


@pytest.mark.parametrize("B,S,Hq,Hkv,D,page,dtype,layout,R,inter,past", APPEND)
def test_append_writes_the_definition(ops, B, S, Hq, Hkv, D, page, dtype, layout, R, inter, past):
    g = _gen(B * 1000 + S)
    n = torch.randint(past // 2, past + 1, (B,), generator=g, dtype=torch.int32)
    per = -(-(past + S) // page)
    table, pages = _table(g, B, per)
    pool = _garbage_pool(g, pages, Hkv, page, D)
    shape = (lambda H: (B, H, S, D)) if layout == "HND" else (lambda H: (B, S, H, D))
    q, k, v = (_randn(g, *shape(H), dtype=dtype) for H in (Hq, Hkv, Hkv))
    v[..., : D // 2] *= 30
    k.view(-1)[:D] = 0.375                       # a constant group: scale 0
    cos = sin = None
    if R:
        a = torch.arange(past + S).double()[:, None] * 10000.0 ** (-torch.arange(0, R, 2).double() / R)
        cos, sin = a.cos().float(), a.sin().float()
    dpool = pool.cuda()
    c = (lambda t: None if t is None else t.cuda())
    qo = ops.kv4_append(dpool, table.cuda(), n.cuda(), k.cuda(), v.cuda(), q=q.cuda(), cos=c(cos), sin=c(sin),
                        interleaved=inter, tensor_layout=layout)
    kr, vr = ops.kv4_read(dpool, table.cuda(), n.cuda(), S, dtype=torch.float32, tensor_layout=layout)
    hnd = (lambda x: x) if layout == "HND" else (lambda x: x.transpose(1, 2))
    at = n.long()[:, None] + torch.arange(S)
    turn = (lambda x: O.rotate(x, cos[at][:, None], sin[at][:, None], inter)) if R else (lambda x: x.float())
    assert torch.equal(hnd(qo.cpu()), turn(hnd(q)).to(dtype))
    for got, want in ((kr, turn(hnd(k))), (vr, hnd(v).float())):
        assert torch.equal(hnd(got.cpu()), O.dequantise(*O.quantise(want)))
    # the records byte by byte, and nothing else written
    after = dpool.cpu()
    for b in range(B):
        for h in range(Hkv):
            full = O.decode(after, table[b], h, int(n[b]) + S)
            assert torch.equal(full[0][int(n[b]):], hnd(kr.cpu())[b, h])
            assert torch.equal(full[1][int(n[b]):], hnd(vr.cpu())[b, h])
    seen = torch.zeros(pages * page, dtype=torch.bool)
    for b in range(B):
        i = at[b]
        seen[table[b].long()[i // page] * page + i % page] = True
    same = lambda lo, hi, row: (after[..., lo:hi].reshape(pages, Hkv, page // 16, 16, row).transpose(1, 2)
                                .reshape(pages, page // 16, Hkv, 16, row).transpose(2, 3).reshape(pages * page, -1)
                                == pool[..., lo:hi].reshape(pages, Hkv, page // 16, 16, row).transpose(1, 2)
                                .reshape(pages, page // 16, Hkv, 16, row).transpose(2, 3).reshape(pages * page, -1))
    for lo, hi, row in ((0, 8 * D, D // 2), (8 * D, 16 * D, D // 2), (16 * D, 17 * D, D // 16), (17 * D, 18 * D, D // 16)):
        assert same(lo, hi, row)[~seen].all()
    # other types of the same values
    for dt in (BF, HF):
        k16, _ = ops.kv4_read(dpool, table.cuda(), n.cuda(), S, dtype=dt, tensor_layout=layout)
        assert torch.equal(k16.cpu(), kr.cpu().to(dt))


def test_append_counts_positions_and_strides(ops):
    g = _gen(5)
    B, S, H, D, page = 3, 20, 2, 64, 16
    table, pages = _table(g, B, 3)
    pool = _garbage_pool(g, pages, H, page, D)
    big = _randn(g, B, S * 2, H, 3 * D).cuda()           # k, v, q interleaved in one projection, every second token
    q, k, v = (big[:, ::2, :, i * D:(i + 1) * D] for i in range(3))
    cos, sin = torch.rand((50, 16), generator=g), torch.rand((50, 16), generator=g)
    pos = torch.randint(0, 50, (B, S), generator=g)      # int64, out of order
    counts, n = torch.tensor([0, 20, 7]), torch.tensor([4, 16, 0])
    dpool = pool.cuda()
    qo = ops.kv4_append(dpool, table.cuda(), n.cuda(), k, v, q=q, cos=cos.cuda(), sin=sin.cuda(), positions=pos.cuda(),
                        counts=counts.cuda(), tensor_layout="NHD")
    hnd = lambda x: x.transpose(1, 2).cpu()
    want_q = O.rotate(hnd(q), cos[pos][:, None], sin[pos][:, None], False).to(BF)
    assert torch.equal(hnd(qo), want_q)
    wk = O.dequantise(*O.quantise(O.rotate(hnd(k), cos[pos][:, None], sin[pos][:, None], False)))
    wv = O.dequantise(*O.quantise(hnd(v)))
    after = dpool.cpu()
    for b in range(B):
        c, s = int(counts[b]), int(n[b])
        for h in range(H):
            fk, fv = O.decode(after, table[b], h, s + c)
            assert torch.equal(fk[s:], wk[b, h, :c]) and torch.equal(fv[s:], wv[b, h, :c])
    used = {int(table[b, (int(n[b]) + t) // page]) for b in range(B) for t in range(int(counts[b]))}
    for p in set(range(pages)) - used:
        assert torch.equal(after[p], pool[p])


def test_append_special_values(ops):
    """Groups with NaN or infinity read as NaN; tiny and huge finite groups, zeros and constants survive."""
    D = 128
    k = torch.zeros((1, 1, 8, D), dtype=BF)
    g = _gen(9)
    k[0, 0, 1] = _randn(g, D)
    k[0, 0, 1, 3] = math.nan
    k[0, 0, 2, 70] = math.inf
    k[0, 0, 3, 0] = -math.inf
    k[0, 0, 4] = _randn(g, D) * 2.0 ** -130          # scale below the least normal float: flushed
    k[0, 0, 5] = _randn(g, D) * 2.0 ** 120
    k[0, 0, 6] = 7.0
    k[0, 0, 7, :64] = 2.0 ** -100 * _randn(g, 64)
    table, pool = torch.zeros((1, 1), dtype=torch.int32), ops.kv4_pool(1, 1, D, 16)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv4_append(pool, table.cuda(), zero, k.cuda(), k.cuda())
    kr, vr = ops.kv4_read(pool, table.cuda(), None, 8, dtype=torch.float32)
    want = O.dequantise(*O.quantise(k))
    for got in (kr.cpu(), vr.cpu()):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(got.nan_to_num(), want.nan_to_num())
    assert want[0, 0, 1, :64].isnan().all() and not want[0, 0, 1, 64:].isnan().any()
    assert want[0, 0, 2, 64:].isnan().all() and want[0, 0, 3, :64].isnan().all()
    assert torch.equal(kr.cpu()[0, 0, 6], torch.full((D,), 7.0))


def test_tokens_without_a_page_are_reported(ops):
    """An entry outside the pool, an index past the table and a position past the rotation table set the error
    bit; the other tokens of the call are written."""
    D, page = 64, 16
    g = _gen(3)
    table = torch.tensor([[0, 7], [-1, 1]], dtype=torch.int32)     # 3 pages in the pool
    pool = ops.kv4_pool(3, 1, D, page)
    k = _randn(g, 2, 1, 18, D).cuda()
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    ops.kv4_append(pool, table.cuda(), zero, k, k)
    assert ops.error_word(0, clear=True) == 0x80
    got, _ = ops.kv4_read(pool, table.cuda(), None, 18, dtype=torch.float32)
    assert ops.error_word(0, clear=True) == 0x80
    want = O.dequantise(*O.quantise(k.cpu()))
    assert torch.equal(got.cpu()[0, 0, :16], want[0, 0, :16]) and torch.equal(got.cpu()[1, 0, 16:], want[1, 0, 16:])
    assert not got[0, 0, 16:].any() and not got[1, 0, :16].any()
    ops.kv4_append(pool, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), torch.tensor([15], device="cuda"),
                   k[:1, :, :2], k[:1, :, :2])                     # second token past the table's width
    assert ops.error_word(0, clear=True) == 0x80
    cos = torch.ones((4, 16), device="cuda")
    ops.kv4_append(pool, torch.zeros((1, 1), dtype=torch.int32, device="cuda"), zero[:1], k[:1, :, :6], k[:1, :, :6],
                   cos=cos, sin=cos)                               # positions 4 and 5 have no row
    assert ops.error_word(0, clear=True) == 0x80


# ---------------------------------------------------------------------------
# attention over the cache
# ---------------------------------------------------------------------------
def _check(got, want, dtype, D, bits):
    out, mass, reach = want
    tol = O.attention_tolerance(out, mass, reach, dtype, D, operand_bits=bits)
    err = (got.cpu().double() - out).abs()
    assert got.isfinite().all()
    worst = (err / tol.clamp_min(1e-30)).max()
    assert bool((err <= tol).all()), f"error up to {float(worst):.2f} of the bound"


KV4 = [  # lengths, Sq, Hq, Hkv, D, page, dtype, layout, causal, window, sinks
    ([1], 1, 1, 1, 128, 16, BF, "HND", True, 0, 0),
    ([1, 17, 200], 1, 4, 2, 64, 64, HF, "NHD", True, 0, 0),
    ([700, 33, 511], 1, 7, 1, 128, 64, BF, "HND", True, 0, 0),
    ([260, 1023], 1, 32, 4, 128, 32, HF, "NHD", True, 100, 4),
    ([1500], 1, 40, 2, 64, 128, BF, "HND", True, 64, 0),
    ([300, 129], 5, 8, 2, 128, 64, BF, "NHD", True, 0, 0),
    ([90, 400], 3, 6, 2, 64, 16, HF, "HND", False, 50, 20),
    ([64, 640], 16, 16, 2, 128, 256, BF, "HND", True, 33, 1),
    ([200], 200, 3, 3, 64, 64, BF, "NHD", True, 0, 0),
    ([777, 300], 130, 14, 2, 128, 64, BF, "HND", True, 0, 0),
    ([500, 450], 257, 4, 4, 64, 128, HF, "NHD", False, 200, 30),
    ([900], 300, 2, 1, 128, 32, HF, "HND", True, 70, 10),
    ([40, 1030], 40, 28, 4, 128, 16, BF, "NHD", False, 0, 0),
    ([600, 90], 7, 8, 2, 128, 64, HF, "HND", True, 0, 0),
    ([600, 90], 7, 8, 2, 128, 64, BF, "HND", True, 0, 0),
    ([600, 90], 6, 8, 2, 128, 64, HF, "NHD", True, 200, 7),
    ([333], 32, 3, 3, 64, 32, HF, "HND", False, 0, 0),
]


@pytest.mark.parametrize("lengths,Sq,Hq,Hkv,D,page,dtype,layout,causal,window,sinks", KV4)
def test_attention_over_the_cache(ops, lengths, Sq, Hq, Hkv, D, page, dtype, layout, causal, window, sinks):
    g = _gen(sum(lengths) + Sq)
    B = len(lengths)
    pool, table, n = _filled(ops, g, B, Hkv, D, page, lengths)
    q = _randn(g, B, Hq, Sq, D, dtype=dtype)
    dq = q.cuda() if layout == "HND" else q.transpose(1, 2).contiguous().cuda()
    got = ops.kv4_attention(dq, pool, table.cuda(), n.cuda(), causal=causal, window=window or None, sinks=sinks,
                            tensor_layout=layout)
    assert got.shape == dq.shape and got.dtype == dtype
    got = got if layout == "HND" else got.transpose(1, 2)
    want = O.paged_attention(q, pool.cpu(), table, n, causal=causal, window=window, sinks=sinks)
    _check(got, want, dtype, D, 11)
    again = ops.kv4_attention(dq, pool, table.cuda(), n.cuda(), causal=causal, window=window or None, sinks=sinks,
                              tensor_layout=layout)
    assert torch.equal(again, got if layout == "HND" else got.transpose(1, 2))    # repeatable bit for bit


@pytest.mark.parametrize("Sq", [1, 6, 140])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_rows_that_see_nothing(ops, D, Sq):
    """Empty sequences, sequences shorter than the queries and short q_lengths: zeros there, the rest unharmed."""
    g = _gen(Sq)
    lengths = [0, 5, 300, 300]
    pool, table, n = _filled(ops, g, 4, 2, D, 64, lengths)
    q = _randn(g, 4, 4, Sq, D)
    ql = torch.tensor([Sq, Sq, 0, max(1, Sq - 3)])
    got = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda(), q_lengths=ql.cuda())
    want = O.paged_attention(q, pool.cpu(), table, n, q_lengths=ql)
    _check(got, want, BF, D, 11)
    got = got.cpu()
    assert not got[0].any() and not got[2].any() and not got[3, :, int(ql[3]):].any()
    if Sq > 5:
        assert not got[1, :, : Sq - 5].any()


@pytest.mark.parametrize("Sq,Hq", [(1, 8), (4, 32), (150, 2)])
def test_attention_large_logits_and_scales(ops, Sq, Hq):
    """Keys that dominate late in the sequence, values over many orders of magnitude, big and small queries."""
    g = _gen(31)
    D, L, page = 128, 700, 64
    table, pages = _table(g, 1, -(-L // page))
    pool = _garbage_pool(g, pages, 2, page, D).cuda()
    k, v = _randn(g, 1, 2, L, D), _randn(g, 1, 2, L, D)
    k[:, :, 600:] *= 6
    v[:, :, ::3] *= 64
    v[:, :, 1::3] *= 2.0 ** -6
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv4_append(pool, table.cuda(), zero, k.cuda(), v.cuda())
    q = _randn(g, 1, Hq, Sq, D)
    q[:, 0] *= 2.0 ** 7
    q[:, 1] *= 2.0 ** -20
    n = torch.tensor([L], dtype=torch.int32)
    got = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda(), sm_scale=0.05)
    _check(got, O.paged_attention(q, pool.cpu(), table, n, scale=0.05), BF, D, 11)


def test_attention_nan_and_infinity_stay_where_they_are_seen(ops):
    """A query with NaN, and a cached token whose values are NaN: only rows that see them are NaN."""
    g = _gen(8)
    D, L = 64, 400
    pool, table, n = _filled(ops, g, 1, 1, D, 64, [L])
    k = _randn(g, 1, 1, 1, D)
    bad = torch.full_like(k, math.nan)
    ops.kv4_append(pool, table.cuda(), torch.tensor([10], device="cuda"), k.cuda(), bad.cuda())   # token 10's value
    q = _randn(g, 1, 4, 1, D)
    q[0, 2, 0, 5] = math.nan
    far = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda(), window=128, sinks=4).cpu()
    assert far[0, [0, 1, 3]].isfinite().all() and far[0, 2].isnan().all()
    near = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda()).cpu()
    assert near.isnan().all()


def test_attention_out_of_range_metadata_is_reported(ops):
    g = _gen(4)
    pool, table, n = _filled(ops, g, 2, 1, 64, 16, [64, 64])
    q = _randn(g, 2, 1, 1, 64).cuda()
    broken = table.clone()
    broken[0, 1] = 99
    got = ops.kv4_attention(q, pool, broken.cuda(), n.cuda())
    assert ops.error_word(0, clear=True) == 0x80 and got.isfinite().all()
    good = ops.kv4_attention(q, pool, table.cuda(), n.cuda())
    assert torch.equal(got[1], good[1])
    too_long = torch.tensor([64, 16 * table.shape[1] + 1], dtype=torch.int32)
    ops.kv4_attention(q, pool, table.cuda(), too_long.cuda())
    assert ops.error_word(0, clear=True) == 0x80


def test_attention_max_length_hint_out_and_other_stream(ops):
    g = _gen(12)
    pool, table, n = _filled(ops, g, 2, 2, 128, 64, [500, 90])
    q = _randn(g, 2, 4, 2, 128).cuda()
    want = O.paged_attention(q.cpu(), pool.cpu(), table, n)
    for hint in (None, 500, 100000):
        _check(ops.kv4_attention(q, pool, table.cuda(), n.cuda(), max_length=hint), want, BF, 128, 11)
    out = torch.zeros((2, 4, 2, 256), dtype=BF, device="cuda")[..., 64:192]
    assert ops.kv4_attention(q, pool, table.cuda(), n.cuda(), out=out) is out
    _check(out, want, BF, 128, 11)
    odd = torch.zeros((2, 4, 2, 131), dtype=BF, device="cuda")[..., 1:129]       # not aligned: written through a copy
    assert ops.kv4_attention(q, pool, table.cuda(), n.cuda(), out=odd) is odd
    assert torch.equal(odd, out)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = ops.kv4_attention(q, pool, table.cuda(), n.cuda())
    st.synchronize()
    assert torch.equal(again, out)


def test_long_cache_offsets(ops):
    """A pool whose byte offsets pass 32 bits: the pages in use are the last ones."""
    D, H, page = 128, 8, 256
    per = H * page * 18 * D // 16
    pages = (1 << 32) // per + 40
    pool = torch.empty((pages, H, page // 16, 18 * D), dtype=torch.uint8, device="cuda")
    g = _gen(2)
    L = 1100
    table = torch.arange(pages - 5, pages, dtype=torch.int32)[None].contiguous()
    k, v = _randn(g, 1, H, L, D), _randn(g, 1, H, L, D)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    ops.kv4_append(pool, table.cuda(), zero, k.cuda(), v.cuda())
    kr, _ = ops.kv4_read(pool, table.cuda(), None, L, dtype=torch.float32)
    assert torch.equal(kr.cpu(), O.dequantise(*O.quantise(k)))
    small, n = pool[pages - 5:].cpu(), torch.tensor([L], dtype=torch.int32)
    for Sq in (1, 130):
        q = _randn(g, 1, H, Sq, D)
        got = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda())
        _check(got, O.paged_attention(q, small, table - (pages - 5), n), BF, D, 11)


# ---------------------------------------------------------------------------
# window attention
# ---------------------------------------------------------------------------
WINDOW = [  # B, Sq, Sk, Hq, Hkv, D, dtype, layout, causal, window, sinks, kv_lengths
    (1, 1, 1, 1, 1, 64, BF, "HND", True, 0, 0, None),
    (2, 1, 300, 8, 2, 128, HF, "NHD", True, 0, 0, None),
    (2, 131, 131, 4, 2, 64, HF, "HND", True, 64, 4, [131, 60]),
    (1, 257, 257, 7, 1, 128, BF, "NHD", True, 0, 0, None),
    (1, 300, 300, 2, 2, 128, HF, "HND", False, 0, 0, None),
    (2, 200, 513, 6, 3, 64, BF, "NHD", True, 100, 10, None),
    (1, 640, 640, 1, 1, 128, BF, "HND", True, 130, 70, None),
    (1, 640, 640, 3, 1, 64, HF, "HND", True, 1, 0, None),
    (1, 129, 700, 5, 5, 128, BF, "NHD", False, 200, 1, None),
    (3, 100, 40, 2, 1, 64, BF, "HND", True, 16, 2, None),           # more queries than keys
    (4, 150, 300, 4, 4, 128, HF, "HND", False, 0, 0, [0, 1, 128, 300]),
    (1, 1000, 1000, 16, 2, 64, BF, "NHD", True, 256, 300, None),
]


@pytest.mark.parametrize("B,Sq,Sk,Hq,Hkv,D,dtype,layout,causal,window,sinks,kvl", WINDOW)
def test_window_attention(ops, B, Sq, Sk, Hq, Hkv, D, dtype, layout, causal, window, sinks, kvl):
    g = _gen(Sq * 7 + Sk)
    q, k, v = (_randn(g, B, H, S, D, dtype=dtype) for H, S in ((Hq, Sq), (Hkv, Sk), (Hkv, Sk)))
    n = None
    if kvl is not None:
        n = torch.tensor(kvl, dtype=torch.int32)
        for b in range(B):   # what lies past the end is garbage
            k[b, :, kvl[b]:] = math.nan
            v[b, :, kvl[b]:] = math.inf
    lay = (lambda t: t.cuda()) if layout == "HND" else (lambda t: t.transpose(1, 2).contiguous().cuda())
    args = dict(causal=causal, window=window or None, sinks=sinks, kv_lengths=None if n is None else n.cuda(),
                tensor_layout=layout)
    got = ops.window_attention(lay(q), lay(k), lay(v), **args)
    again = ops.window_attention(lay(q), lay(k), lay(v), **args)
    assert torch.equal(got, again)
    got = got if layout == "HND" else got.transpose(1, 2)
    want = O.window_attention(q, k, v, kv_lengths=n, causal=causal, window=window, sinks=sinks)
    _check(got, want, dtype, D, 8 if dtype is BF else 11)
    # rows without a visible key are exactly zero
    none = want[1].sum(-1) == 0
    assert not got.cpu()[none].any()


def test_window_attention_large_logits_and_rescales(ops):
    g = _gen(77)
    q, k, v = (_randn(g, 1, 2, 520, 128) for _ in range(3))
    k = k * (torch.arange(520)[:, None] / 60).to(BF)        # the maximum grows tile after tile
    q[:, 1] *= 16
    for kw in ({}, {"window": 200, "sinks": 130}):
        got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), **kw)
        _check(got, O.window_attention(q, k, v, **kw), BF, 128, 8)


def test_window_attention_strides_and_streams(ops):
    g = _gen(21)
    B, S, H, D = 2, 200, 3, 64
    packed = _randn(g, B, S, H, 3 * D + 5).cuda()            # unaligned slices of one projection
    q, k, v = (packed[..., 1 + i * D:1 + (i + 1) * D] for i in range(3))
    got = ops.window_attention(q, k, v, window=50, sinks=3, tensor_layout="NHD")
    hnd = lambda x: x.transpose(1, 2).cpu()
    _check(got.transpose(1, 2), O.window_attention(hnd(q), hnd(k), hnd(v), window=50, sinks=3), BF, D, 8)
    one = _randn(g, B, 1, H, D).cuda().expand(B, S, H, D)    # broadcast tokens
    got = ops.window_attention(q, one, one, tensor_layout="NHD")
    _check(got.transpose(1, 2), O.window_attention(hnd(q), hnd(one), hnd(one)), BF, D, 8)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        again = ops.window_attention(q, one, one, tensor_layout="NHD")
    st.synchronize()
    assert torch.equal(again, got)


def test_window_attention_no_keys(ops):
    q = torch.randn((2, 2, 9, 64), device="cuda", dtype=BF)
    k = torch.empty((2, 1, 0, 64), device="cuda", dtype=BF)
    assert not ops.window_attention(q, k, k).any()
    assert ops.window_attention(q[:, :, :0], k, k).shape == (2, 2, 0, 64)


# ---------------------------------------------------------------------------
# together
# ---------------------------------------------------------------------------
def test_prompt_then_tokens_matches_one_long_call(ops):
    """Chunks and single tokens through the cache see what one call over the whole sequence sees (same cache)."""
    g = _gen(99)
    B, Hq, H, D, page, L = 2, 8, 2, 128, 64, 300
    table, pages = _table(g, B, -(-L // page))
    pool, dt = ops.kv4_pool(pages, H, D, page), table.cuda()
    q, k, v = (_randn(g, B, h, L, D).cuda() for h in (Hq, H, H))
    done, outs = 0, []
    for step in (200, 1, 1, 3, 60, 1, 34):
        n0 = torch.full((B,), done, dtype=torch.int32, device="cuda")
        ops.kv4_append(pool, dt, n0, k[:, :, done:done + step], v[:, :, done:done + step])
        done += step
        outs.append(ops.kv4_attention(q[:, :, done - step:done], pool, dt, n0 + step, window=90, sinks=5))
    n = torch.full((B,), L, dtype=torch.int32)
    want = O.paged_attention(q.cpu(), pool.cpu(), table, n, window=90, sinks=5)
    _check(torch.cat(outs, 2), want, BF, D, 11)


@pytest.mark.parametrize("H,Sq,Sk,causal", [(160, 20, 1100, True), (80, 130, 3200, False), (100, 40, 4100, True)])
def test_items_cut_after_the_full_waves(ops, H, Sq, Sk, causal):
    """One item a head: 12 of 160 in equal shares; 80 and 100 in a long and a short share each."""
    g = _gen(H)
    q, k, v = _randn(g, 1, H, Sq, 64), _randn(g, 1, H, Sk, 64), _randn(g, 1, H, Sk, 64)
    got = ops.window_attention(q.cuda(), k.cuda(), v.cuda(), causal=causal)
    assert torch.equal(got, ops.window_attention(q.cuda(), k.cuda(), v.cuda(), causal=causal))
    _check(got, O.window_attention(q, k, v, causal=causal), BF, 64, 8)


def test_items_cut_over_the_cache(ops):
    g = _gen(5)
    lengths = [3300, 3111]
    pool, table, n = _filled(ops, g, 2, 40, 64, 64, lengths, dtype=HF)
    q = _randn(g, 2, 40, 40, 64, dtype=HF)
    got = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda())
    _check(got, O.paged_attention(q, pool.cpu(), table, n), HF, 64, 11)


def test_direct_calls_equal_the_wrappers(ops, monkeypatch):
    """Arguments that the extension takes give the same through the wrappers' own code."""
    from vc_b200 import _native as N
    g = _gen(8)
    B, Hq, H, S, D = 2, 6, 2, 70, 128
    table = torch.randperm(8, generator=g).to(torch.int32).view(2, 4).cuda()
    n = torch.tensor([3, 40], dtype=torch.int32, device="cuda")
    cos, sin = torch.rand((256, 32), generator=g).cuda(), torch.rand((256, 32), generator=g).cuda()
    counts = torch.tensor([70, 9], dtype=torch.int32, device="cuda")
    pos = torch.randint(0, 256, (B, S), generator=g, dtype=torch.int32).cuda()
    taken = []

    def run(layout):
        shape = (lambda h: (B, h, S, D)) if layout == "HND" else (lambda h: (B, S, h, D))
        g2 = _gen(9)
        q, k, v = (_randn(g2, *shape(h)).cuda() for h in (Hq, H, H))
        pool = ops.kv4_pool(8, H, D, 64)
        out = [ops.kv4_append(pool, table, n, k, v, q=q, cos=cos, sin=sin, tensor_layout=layout, interleaved=True),
               ops.kv4_append(pool, table, n, k, v, positions=pos, counts=counts, cos=cos, sin=sin, tensor_layout=layout),
               *ops.kv4_read(pool, table, n, 60, dtype=torch.float16, tensor_layout=layout),
               *ops.kv4_read(pool, table, None, 60, tensor_layout=layout),
               ops.kv4_attention(q, pool, table, n + S, tensor_layout=layout),
               ops.kv4_attention(q, pool, table, n + S, q_lengths=counts, causal=False, window=30, sinks=5, sm_scale=0.05,
                                 max_length=120, tensor_layout=layout),
               ops.window_attention(q, k, v, tensor_layout=layout),
               ops.window_attention(q, k, v, window=20, sinks=3, causal=False, kv_lengths=counts, sm_scale=0.2,
                                    tensor_layout=layout), pool]
        return out

    class Counting:
        def __getattr__(self, name):
            fn = getattr(real, name)

            def call(*a):
                r = fn(*a)
                taken.append(r is not NotImplemented)
                return r
            return call

    class Refusing:
        def __getattr__(self, name):
            return lambda *a: NotImplemented

    real = N.calls()
    for layout in ("HND", "NHD"):
        monkeypatch.setattr(N, "calls", Counting)
        a = run(layout)
        monkeypatch.setattr(N, "calls", Refusing)
        b = run(layout)
        for x, y in zip(a, b):
            assert (x is None and y is None) or (x.dtype == y.dtype and x.shape == y.shape and torch.equal(x, y))
    assert len(taken) == 16 and all(taken)
    ops.error_word(0, clear=True)   # (the 120-token bound cut a sequence)


def test_refusals_on_the_device(ops):
    g = _gen(1)
    pool = ops.kv4_pool(4, 2, 64, 16)
    table = torch.zeros((1, 2), dtype=torch.int32, device="cuda")
    n = torch.zeros(1, dtype=torch.int32, device="cuda")
    k = _randn(g, 1, 2, 4, 64).cuda()
    q = _randn(g, 1, 4, 4, 64).cuda()
    bad = [
        lambda: ops.kv4_append(pool, table, n, k.float(), k.float()),
        lambda: ops.kv4_append(pool, table, n, k, k[:, :1]),
        lambda: ops.kv4_append(pool, table, n, k, k.half()),
        lambda: ops.kv4_append(pool, table, n, k, k, q=q[:, :3]),
        lambda: ops.kv4_append(pool, table, n[:0], k, k),
        lambda: ops.kv4_append(pool, table, n.float(), k, k),
        lambda: ops.kv4_append(pool, table.long(), n, k, k),
        lambda: ops.kv4_append(pool, table.cpu(), n, k, k),
        lambda: ops.kv4_append(pool, table, n, k, k, cos=torch.ones((4, 4), device="cuda")),
        lambda: ops.kv4_append(pool, table, n, k, k, cos=torch.ones((4, 4), device="cuda"), sin=torch.ones((4, 4), device="cuda")),
        lambda: ops.kv4_append(pool, table, n, k, k, cos=torch.ones((4, 40), device="cuda"), sin=torch.ones((4, 40), device="cuda")),
        lambda: ops.kv4_append(pool[:, :, :, :100], table, n, k, k),
        lambda: ops.kv4_append(pool, table, n, k.requires_grad_(True), k),
        lambda: ops.kv4_read(pool, table, n, -1),
        lambda: ops.kv4_read(pool, table, n, 1, dtype=torch.float64),
        lambda: ops.kv4_attention(q[:, :3], pool, table, n),
        lambda: ops.kv4_attention(q, pool, table, n, window=0),
        lambda: ops.kv4_attention(q, pool, table, n, sinks=-1),
        lambda: ops.kv4_attention(q, pool, table, n, sm_scale=math.inf),
        lambda: ops.kv4_attention(q, pool, table, n, tensor_layout="SHD"),
        lambda: ops.kv4_attention(q, pool, table, n, out=q[:, :2]),
        lambda: ops.kv4_attention(q, pool, table, n, q_lengths=n.float()),
        lambda: ops.window_attention(q, k.detach()[..., :32], k.detach()[..., :32]),
        lambda: ops.window_attention(q[:, :3], k.detach(), k.detach()),
        lambda: ops.window_attention(q[0], k.detach()[0], k.detach()[0]),
        lambda: ops.window_attention(q, k.detach(), k.detach(), kv_lengths=n[:0]),
        lambda: ops.window_attention(q, k.detach(), k.detach(), causal=None),
        lambda: ops.kv4_pool(4, 2, 96),
        lambda: ops.kv4_pool(4, 2, 64, 24),
    ]
    for i, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i} was not refused")


@pytest.mark.parametrize("Sq,page", [(1, 16), (5, 16), (40, 32), (300, 16), (1, 128)])
def test_pages_that_no_query_sees_may_be_missing(ops, Sq, page):
    """Behind the window and past the sinks the table may say anything."""
    g = _gen(Sq + page)
    D, L, window, sinks = 128, 900, 200, 20
    pool, table, n = _filled(ops, g, 1, 2, D, page, [L])
    q = _randn(g, 1, 8, Sq, D)
    full = ops.kv4_attention(q.cuda(), pool, table.cuda(), n.cuda(), window=window, sinks=sinks)
    holes = table.clone()
    lo = L - Sq - window + 1
    holes[0, -(-sinks // page): lo // page] = -1
    assert (holes != table).sum() > 1
    assert torch.equal(ops.kv4_attention(q.cuda(), pool, holes.cuda(), n.cuda(), window=window, sinks=sinks), full)


def test_rolling_cache(ops):
    """KV4Cache: pages come and go, ragged appends, and the results are those of a cache that keeps everything."""
    from vc_b200.kv_cache import KV4Cache
    g = _gen(41)
    B, H, Hq, D, window, sinks = 2, 2, 4, 64, 48, 10
    kw = dict(page_size=16, window=window, sinks=sinks)
    small = KV4Cache(B, H, D, pages=16, max_tokens=400, **kw)
    large = KV4Cache(B, H, D, pages=60, max_tokens=400, **kw)
    freed, lengths = 0, [0, 0]
    for step, counts in ((40, None), (20, [20, 3]), (1, None), (33, [0, 33]), (1, None), (30, None), (30, [30, 29])):
        k, v, q = (_randn(g, B, h, step, D).cuda() for h in (H, H, Hq))
        for c in (small, large):
            assert c.append(k, v, q, counts=counts) is not None
        counts = counts or [step] * B
        lengths = [a + b for a, b in zip(lengths, counts)]
        assert small.lengths.tolist() == lengths
        ql = torch.tensor(counts, device="cuda")
        assert torch.equal(small.attend(q, q_lengths=ql), large.attend(q, q_lengths=ql))
        freed += small.trim()
    assert freed > 0 and small.free_pages + freed > 0
    before = small.free_pages
    with pytest.raises(RuntimeError, match="pages needed"):
        small.append(*(_randn(g, B, H, 250, D).cuda() for _ in range(2)))
    assert small.free_pages == before and small.lengths.tolist() == lengths
    with pytest.raises(RuntimeError, match="max_tokens"):
        large.append(*(_randn(g, B, H, 390, D).cuda() for _ in range(2)))
    small.drop(0)
    assert small.lengths.tolist() == [0, lengths[1]] and small.free_pages > before
    with pytest.raises(ValueError, match="counts"):
        small.append(k, v, counts=[1])


def test_streaming_example_runs(ops):
    """The example's stages are near exact attention: the prompt to BF16 rounding, the cache to 4 bits."""
    from vc_attention.streaming import run
    reports = run(400, (130, 8, 1), heads=8, kv_heads=2, window=200, sinks=6)
    assert [r["tokens"] for r in reports] == [400, 130, 8, 1]
    assert reports[0]["rel_l2"] < 2.0 ** -6
    assert all(r["rel_l2"] < 0.25 for r in reports[1:]) and sum(r["pages_freed"] for r in reports) > 0
