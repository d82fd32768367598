"""The cache and window operators as they are measured: cases, inputs, plain
forms and 64-bit results.

Three families, called in turn by a generator that keeps its keys and values
in a paged 4-bit cache:

* ``append``  -- rotate new K (and Q) by position, quantise K/V to 4 bits,
  write them to the cache's pages, and read back the values they stand for;
* ``attend``  -- attention of the newest tokens of each sequence over the
  cache (one token: decoding; a few: drafts; many: a chunk);
* ``window``  -- attention over 16-bit K/V with a sliding window and a few
  first tokens that stay visible.

The cache ("pool") is ``uint8 [pages, kv_heads, page_size / 16, 18 * D]``.  A
record holds 16 tokens of one head: K codes (16 x D/2 bytes, channel 2i in the
low four bits), V codes alike, then for K and for V a (scale, minimum) pair of
bfloat16 per token and 64 channels.
"""
import math
import os
import sys

import torch

own = False

GROUP = 64   # channels that share a scale and a minimum
BLOCK = 16   # tokens of a record
TINY = 2.0 ** -126
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}

# head counts that occur together: (query heads, kv heads)
HEADS = [(28, 4), (32, 8), (24, 8), (24, 24), (8, 8), (40, 8), (16, 2), (2, 1)]


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def _append(name, B, S, past, heads, D, dtype, layout, page, style="half", rotary=1.0):
    return {"name": name, "op": "append", "B": B, "S": S, "past": past, "hq": heads[0], "hkv": heads[1], "D": D,
            "dtype": dtype, "layout": layout, "page": page, "interleaved": style == "interleaved", "rotary": rotary}


def _attend(name, B, Sq, length, ragged, heads, D, dtype, layout, page, causal=True, window=0, sinks=0):
    return {"name": name, "op": "attend", "B": B, "Sq": Sq, "len": length, "ragged": ragged, "hq": heads[0],
            "hkv": heads[1], "D": D, "dtype": dtype, "layout": layout, "page": page, "causal": causal,
            "window": window, "sinks": sinks}


def _window(name, B, Sq, Sk, heads, D, dtype, layout, causal=True, window=0, sinks=0, ragged=False):
    return {"name": name, "op": "window", "B": B, "Sq": Sq, "Sk": Sk, "hq": heads[0], "hkv": heads[1], "D": D,
            "dtype": dtype, "layout": layout, "causal": causal, "window": window, "sinks": sinks, "ragged": ragged}


def listed():
    return [
        # one new token of one sequence: the smallest call of a decoding loop, all latency
        _append("append_1x1", 1, 1, 4000, (32, 8), 128, "bf16", "HND", 64),
        # one token for each of many ragged sequences, small pages, the other rotation style
        _append("append_96x1", 96, 1, 16000, (24, 8), 64, "f16", "NHD", 16, "interleaved"),
        # a whole prompt goes into the cache (token-major tensors, as projections leave them)
        _append("append_prompt", 1, 16384, 0, (28, 4), 128, "bf16", "NHD", 64),
        # decoding one long sequence alone: few rows, a long axis to split
        _attend("step_1x37741", 1, 1, 37741, False, (28, 4), 128, "bf16", "HND", 64),
        # decoding a full ragged batch: the ordinary serving step
        _attend("step_64x8192", 64, 1, 8192, True, (32, 8), 128, "bf16", "HND", 64),
        # decoding with a window and sinks: most of each sequence is skipped
        _attend("step_window", 48, 1, 16384, True, (24, 8), 64, "f16", "NHD", 32, True, 1024, 16),
        # a few drafted tokens a sequence, checked in one pass
        _attend("drafts_16x5", 16, 5, 8191, True, (32, 8), 128, "bf16", "HND", 64),
        # a prompt's next chunk over what is already cached
        _attend("chunk_1024", 1, 1024, 16384, False, (28, 4), 128, "bf16", "NHD", 64),
        # a video chunk whose tokens all see one another, the last chunks and the first frame
        _attend("chunk_video", 2, 700, 6300, False, (24, 24), 64, "f16", "HND", 128, False, 4096, 350),
        # a small odd-sized padded batch
        _window("window_131", 2, 131, 131, (2, 1), 64, "f16", "HND", True, 64, 4, True),
        # ordinary prompts, unlimited window (plain causal order)
        _window("causal_4096", 2, 4096, 4096, (28, 4), 128, "bf16", "NHD"),
        # a long prompt under a window with sinks
        _window("window_16384", 1, 16384, 16384, (8, 8), 128, "bf16", "HND", True, 4096, 64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "window"])
    heads, D = rng.choice(HEADS), rng.choice([64, 128])
    dtype, layout, page = rng.choice(["bf16", "f16"]), rng.choice(["HND", "NHD"]), rng.choice([16, 32, 64, 128])
    window, sinks = (0, 0) if rng.random() < 0.4 else (_log(rng, 1, 8192), rng.choice([0, 1, 4, 16, 64, 350]))
    if op == "append":
        B = _log(rng, 1, 128)
        S = _log(rng, 1, max(1, 16384 * 28 // (B * heads[0])))   # at most the listed prompt's rows
        c = _append("", B, S, _log(rng, 1, 8192) - 1, heads, D, dtype, layout, page,
                    rng.choice(["half", "interleaved"]), rng.choice([1.0, 1.0, 0.5]))
    elif op == "attend":
        form = rng.random()
        if form < 0.6:     # decoding and drafts
            B, Sq = _log(rng, 1, 96), rng.choice([1, 1, 1, 2, 3, 5, 8])
            # total cached tokens x kv heads at most those of the largest listed step
            length = _log(rng, max(Sq, 16), max(64, min(100000, 4 * 1024 * 1024 // (B * heads[1]))))
        else:              # chunks: at most the listed chunk's score count
            B, Sq = _log(rng, 1, 4), _log(rng, 9, 2048)
            length = _log(rng, Sq + 1, max(Sq + 2, min(32768, 28 * 1024 * 16384 // (B * heads[0] * Sq))))
        c = _attend("", B, Sq, max(length, Sq), rng.random() < 0.5, heads, D, dtype, layout, page,
                    rng.random() < 0.8, window, sinks)
    else:
        B = _log(rng, 1, 8)
        most = int(math.sqrt(2 * 28 * 4096 * 4096 / (B * heads[0])))
        Sk = _log(rng, 17, max(18, min(16384, most)))
        Sq = Sk if rng.random() < 0.75 else _log(rng, 1, Sk)
        c = _window("", B, Sq, Sk, heads, D, dtype, layout, rng.random() < 0.85, window, sinks, rng.random() < 0.3)
    del c["name"]
    return c


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 1000003 + 17)


def _heads_tensor(g, B, H, S, D, dtype, layout, offset=None):
    """N(0,1) values, with a per-channel offset where a path has one (keys do),
    in the layout that the caller's projections leave."""
    shape = (B, H, S, D) if layout == "HND" else (B, S, H, D)
    x = torch.randn(shape, generator=g, device="cuda")
    if offset is not None:
        x += offset if layout == "HND" else offset.transpose(1, 2)
    return x.to(dtype)


def _key_offset(g, H, D):
    return torch.randn((1, H, 1, D), generator=g, device="cuda")


def _lengths(case, g, most, least):
    B = case["B"]
    if not case["ragged"]:
        return torch.full((B,), most, dtype=torch.int32, device="cuda")
    n = torch.randint(max(least, most // 16), most + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    n[0] = most
    return n


def _paged(case, g, tokens):
    """A pool whose pages hold whatever an earlier user left, and a table of
    scattered pages that covers ``tokens`` tokens of every sequence."""
    B, page = case["B"], case["page"]
    per = -(-tokens // page)
    pages = B * per + 3
    pool = torch.randint(0, 256, (pages, case["hkv"], page // BLOCK, 18 * case["D"]), generator=g, device="cuda",
                         dtype=torch.uint8)
    table = torch.randperm(pages, generator=g, device="cuda")[: B * per].to(torch.int32).view(B, per)
    return pool, table


def _rotation(D, R, tokens):
    """cos and sin by position, the table that a model keeps."""
    inv = 10000.0 ** (-torch.arange(0, R, 2, device="cuda", dtype=torch.float64) / R)
    a = torch.arange(tokens, device="cuda", dtype=torch.float64)[:, None] * inv[None, :]
    return a.cos().float(), a.sin().float()


def prepare(case, seed):
    g = _gen(seed)
    B, D, dt = case["B"], case["D"], DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "append":
        S, R = case["S"], int(D * case["rotary"])
        s["pool"], s["table"] = _paged(case, g, case["past"] + S)
        # sequences have different pasts, and each has room for its new tokens
        s["lengths"] = torch.randint(case["past"] // 2, case["past"] + 1, (B,), generator=g, device="cuda",
                                     dtype=torch.int32)
        s["cos"], s["sin"] = _rotation(D, R, case["past"] + S)
        s["k"] = _heads_tensor(g, B, case["hkv"], S, D, dt, case["layout"], _key_offset(g, case["hkv"], D))
        s["v"] = _heads_tensor(g, B, case["hkv"], S, D, dt, case["layout"])
        s["q"] = _heads_tensor(g, B, case["hq"], S, D, dt, case["layout"])
    elif case["op"] == "attend":
        L = case["len"]
        s["pool"], s["table"] = _paged(case, g, L)
        s["lengths"] = _lengths(case, g, L, case["Sq"])
        off = _key_offset(g, case["hkv"], D)
        step = max(1, (1 << 27) // (B * case["hkv"] * D))   # the cache is filled in pieces
        for a in range(0, L, step):
            n = min(step, L - a)
            k = _heads_tensor(g, B, case["hkv"], n, D, torch.float32, "HND", off)
            v = _heads_tensor(g, B, case["hkv"], n, D, torch.float32, "HND")
            at = torch.arange(a, a + n, device="cuda").expand(B, n)
            _write(s["pool"], s["table"], at, at < s["lengths"][:, None], _quantise(k), _quantise(v))
        s["q"] = _heads_tensor(g, B, case["hq"], case["Sq"], D, dt, case["layout"])
    else:
        s["q"] = _heads_tensor(g, B, case["hq"], case["Sq"], D, dt, case["layout"])
        s["k"] = _heads_tensor(g, B, case["hkv"], case["Sk"], D, dt, case["layout"], _key_offset(g, case["hkv"], D))
        s["v"] = _heads_tensor(g, B, case["hkv"], case["Sk"], D, dt, case["layout"])
        s["kv_lengths"] = _lengths(case, g, case["Sk"], 1) if case["ragged"] else None
    return s


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _quantise(x):
    """(codes uint8 [B,H,S,D], scale and minimum bfloat16 [B,H,S,D/64]) of FP32 values."""
    y = x.unflatten(-1, (-1, GROUP))
    lo, hi = y.amin(-1), y.amax(-1)
    s, m = ((hi - lo) / 15.0).to(torch.bfloat16), lo.to(torch.bfloat16)
    s = torch.where(s.float() < TINY, torch.zeros_like(s), s)
    inv = torch.where(s == 0, torch.zeros_like(s, dtype=torch.float32), 1.0 / s.float())
    u = ((y - m.float().unsqueeze(-1)) * inv.unsqueeze(-1)).round().clamp(0, 15)
    return torch.nan_to_num(u, nan=0.0).to(torch.uint8).flatten(-2), s, m


def _fields(pool):
    """Views of the pool's records: K/V codes [pages,H,blocks,16,D/2] and
    (scale, minimum) [pages,H,blocks,16,D/64,2] bfloat16."""
    D = pool.shape[-1] // 18
    kc, vc, kp, vp = pool.split([8 * D, 8 * D, D, D], -1)
    return (kc.unflatten(-1, (BLOCK, D // 2)), vc.unflatten(-1, (BLOCK, D // 2)),
            kp.view(torch.bfloat16).unflatten(-1, (BLOCK, D // GROUP, 2)),
            vp.view(torch.bfloat16).unflatten(-1, (BLOCK, D // GROUP, 2)))


def _place(pool, table, at):
    """Page, block and slot of tokens ``at`` [B,S], each [B,S,1], and heads [1,1,H]."""
    page = pool.shape[2] * BLOCK
    p = table.long().gather(1, at // page)
    return (p[..., None], torch.arange(pool.shape[1], device=pool.device)[None, None, :],
            (at % page // BLOCK)[..., None], (at % BLOCK)[..., None])


def _write(pool, table, at, keep, kq, vq):
    kc, vc, kp, vp = _fields(pool)
    p, h, b, t = (i.expand(*at.shape, pool.shape[1])[keep] for i in _place(pool, table, at))
    for codes, pairs, (u, s, m) in ((kc, kp, kq), (vc, vp, vq)):
        u, s, m = (x.transpose(1, 2)[keep] for x in (u, s, m))
        codes[p, h, b, t] = u[..., 0::2] | (u[..., 1::2] << 4)
        pairs[p, h, b, t] = torch.stack((s, m), -1)


def _read(pool, table, at):
    """FP32 K and V [B,H,S,D] of tokens ``at`` [B,S]."""
    kc, vc, kp, vp = _fields(pool)
    i = _place(pool, table, at)
    out = []
    for codes, pairs in ((kc, kp), (vc, vp)):
        c, sm = codes[i], pairs[i].float()
        u = torch.stack((c & 15, c >> 4), -1).flatten(-2).float().unflatten(-1, (-1, GROUP))
        out.append((u * sm[..., 0:1] + sm[..., 1:2]).flatten(-2).transpose(1, 2))
    return out


def _rotate(x, cos, sin, interleaved):
    R = 2 * cos.shape[-1]
    y, rest = x[..., :R], x[..., R:]
    a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., : R // 2], y[..., R // 2:])
    p, q = a * cos - b * sin, b * cos + a * sin
    y = torch.stack((p, q), -1).flatten(-2) if interleaved else torch.cat((p, q), -1)
    return torch.cat((y, rest), -1)


def _hnd(x, layout):
    return x if layout == "HND" else x.transpose(1, 2)


def _softmax_product(q, k, v, visible, scale):
    """softmax(scale q k^T) v in FP32 over the visible keys (zero where there
    are none); q [B,Hq,Sq,D], k and v [B,Hkv,L,D], visible [B,1,1,Sq,L]."""
    B, Hq, Sq, D = q.shape
    Hkv = k.shape[1]
    x = q.reshape(B, Hkv, -1, D) @ k.transpose(-1, -2) * scale
    x = x.view(B, Hkv, Hq // Hkv, Sq, -1).masked_fill_(~visible, -math.inf)
    top = x.amax(-1, keepdim=True)
    x = x.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = x.sum(-1, keepdim=True)
    out = x.view(B, Hkv, -1, x.shape[-1]) @ v
    return out.view(B, Hq, Sq, D) / torch.where(total == 0, torch.ones_like(total), total).view(B, Hq, Sq, 1)


def _visible(i, j, length, causal, window, sinks):
    """Which of keys j [L] the queries at positions i [B,Sq] see: [B,Sq,L]."""
    i, ok = i[..., None], j < length[:, None, None]
    if causal:
        ok = ok & (j <= i)
    if window:
        ok = ok & ((j > i - window) | (j < sinks))
    return ok


def _plain(s):
    c = s["case"]
    lay, dt, dev = c["layout"], DTYPES[c["dtype"]], s["q"].device
    if c["op"] == "append":
        at = s["lengths"].long()[:, None] + torch.arange(c["S"], device=dev)
        cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
        q, k = (_rotate(_hnd(s[n], lay).float(), cos, sin, c["interleaved"]) for n in ("q", "k"))
        kq, vq = _quantise(k), _quantise(_hnd(s["v"], lay).float())
        _write(s["pool"], s["table"], at, torch.ones_like(at, dtype=torch.bool), kq, vq)
        kr, vr = _read(s["pool"], s["table"], at)
        return {"q": _hnd(q, lay).to(dt), "k": _hnd(kr, lay).to(dt), "v": _hnd(vr, lay).to(dt)}
    q = _hnd(s["q"], lay).float()
    if c["op"] == "attend":
        L = c["len"]
        j = torch.arange(L, device=dev)
        k, v = _read(s["pool"], s["table"], j.expand(c["B"], L))
        n = s["lengths"].long()
        i = n[:, None] - c["Sq"] + torch.arange(c["Sq"], device=dev)
        # what an earlier user left behind the end of a sequence is not part of it
        v = v.masked_fill(~(j < n[:, None])[:, None, :, None], 0.0)
    else:
        j = torch.arange(c["Sk"], device=dev)
        k, v = _hnd(s["k"], lay).float(), _hnd(s["v"], lay).float()
        n = s["kv_lengths"].long() if s["kv_lengths"] is not None else torch.full((c["B"],), c["Sk"], device=dev)
        i = (c["Sk"] - c["Sq"] + torch.arange(c["Sq"], device=dev)).expand(c["B"], c["Sq"])
    ok = _visible(i, j, n, c["causal"], c["window"], c["sinks"])[:, None, None]
    return _hnd(_softmax_product(q, k, v, ok, c["D"] ** -0.5), lay).to(dt).contiguous()


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
_ops = None


def _own(s):
    global _ops
    if _ops is None:
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "cake-opt-vc_attention_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        from vc_b200 import ops
        _ops = ops
    c = s["case"]
    if c["op"] == "append":
        q = _ops.kv4_append(s["pool"], s["table"], s["lengths"], s["k"], s["v"], q=s["q"], cos=s["cos"], sin=s["sin"],
                            interleaved=c["interleaved"], tensor_layout=c["layout"])
        k, v = _ops.kv4_read(s["pool"], s["table"], s["lengths"], c["S"], dtype=s["q"].dtype,
                             tensor_layout=c["layout"])
        return {"q": q, "k": k, "v": v}
    if c["op"] == "attend":
        return _ops.kv4_attention(s["q"], s["pool"], s["table"], s["lengths"], causal=c["causal"],
                                  window=c["window"] or None, sinks=c["sinks"], tensor_layout=c["layout"])
    return _ops.window_attention(s["q"], s["k"], s["v"], causal=c["causal"], window=c["window"] or None,
                                 sinks=c["sinks"], kv_lengths=s["kv_lengths"], tensor_layout=c["layout"])


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the work of one pass
# ---------------------------------------------------------------------------
def _seen(i, length, causal, window, sinks):
    """How many of ``length`` keys a query at position i sees."""
    hi = min(length, i + 1) if causal else length
    if hi <= 0:
        return 0
    if not window:
        return hi
    lo = max(0, i - window + 1)
    return max(0, hi - lo) + min(sinks, lo, hi)


def work(case):
    c, D = case, case["D"]
    if c["op"] == "append":
        rows, R = c["B"] * c["S"], int(D * c["rotary"])
        # q in and out; k and v in, their records out and in again, their values out; cos and sin
        return {"bytes": rows * (4 * c["hq"] * D + c["hkv"] * (4 * D + 2 * 18 * D // 16 + 4 * D) + 4 * R),
                "flops": rows * (3 * R * (c["hq"] + c["hkv"]) + 16 * D * c["hkv"])}
    # ragged lengths are uniform between a sixteenth and the whole, the first is whole
    share = (17.0 / 32.0 * (c["B"] - 1) + 1.0) / c["B"] if c["ragged"] else 1.0
    L = c["len"] if c["op"] == "attend" else c["Sk"]
    mean = max(1, int(round(L * share)))
    # in a cache the queries are a sequence's last tokens; in tensors padding shortens the keys alone
    end = mean if c["op"] == "attend" else L
    pos = range(end - c["Sq"], end)
    pairs = sum(_seen(i, mean, c["causal"], c["window"], c["sinks"]) for i in pos)
    lo = max(0, pos[0] - c["window"] + 1) if c["window"] else 0
    hi = min(mean, end) if c["causal"] else mean
    keys = max(0, hi - lo) + min(c["sinks"], lo, max(hi, 0))
    per = 18 * D / 16 if c["op"] == "attend" else 4 * D
    return {"bytes": c["B"] * (4 * c["hq"] * c["Sq"] * D + c["hkv"] * keys * per),
            "flops": 4.0 * c["B"] * c["hq"] * pairs * D}


# ---------------------------------------------------------------------------
# 64-bit results
# ---------------------------------------------------------------------------
def _decode64(pool, table, b, n, which):
    """Token values [H, n, D] in 64 bits of K (which = 0) or V (1) of sequence b, from the records' bytes."""
    pages, H, blocks, size = pool.shape
    D = size // 18
    rec = pool[table[b].long()].permute(1, 0, 2, 3).reshape(H, -1, size)[:, : -(-n // BLOCK)]
    code = rec[..., which * 8 * D:(which + 1) * 8 * D].reshape(H, -1, D // 2)[:, :n]
    par = rec[..., 16 * D + which * D: 17 * D + which * D].contiguous().view(torch.bfloat16)
    par = par.reshape(H, -1, D // GROUP, 2)[:, :n].double().repeat_interleave(GROUP, 2)
    u = torch.empty((H, n, D), dtype=torch.float64, device=pool.device)
    u[..., 0::2], u[..., 1::2] = (code % 16).double(), (code // 16).double()
    return u * par[..., 0] + par[..., 1]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    lay, B, D, dev = c["layout"], c["B"], c["D"], s["q"].device
    if c["op"] == "append":
        S, R = c["S"], int(D * c["rotary"])
        at = (s["lengths"].long()[:, None] + torch.arange(S, device=dev)).double()
        ang_c = s["cos"].double()[at.long()][:, None]
        ang_s = s["sin"].double()[at.long()][:, None]
        out = {}
        for name in ("q", "k", "v"):
            x = _hnd(s[name], lay).double().clone()
            if name != "v":
                first, second = (slice(0, R, 2), slice(1, R, 2)) if c["interleaved"] else (slice(0, R // 2), slice(R // 2, R))
                a, b = x[..., first].clone(), x[..., second].clone()
                x[..., first] = a * ang_c - b * ang_s
                x[..., second] = a * ang_s + b * ang_c
            if name != "q":
                y = x.reshape(*x.shape[:-1], D // GROUP, GROUP)
                base = y.min(-1, keepdim=True).values.to(torch.bfloat16).double()
                step = ((y.max(-1, keepdim=True).values - y.min(-1, keepdim=True).values) / 15).to(torch.bfloat16).double()
                n = torch.where(step > 0, (y - base) / step, torch.zeros_like(y)).round().clamp(0, 15)
                x = (n * step + base).reshape(x.shape)
            out[name] = _hnd(x, lay)
        return out
    if work(c)["flops"] > 5e12:
        return None
    scale, G = D ** -0.5, c["hq"] // c["hkv"]
    q = _hnd(s["q"], lay).double()
    out = torch.zeros((B, c["hq"], c["Sq"], D), dtype=torch.float64, device=dev)
    for b in range(B):
        if c["op"] == "attend":
            n = int(s["lengths"][b])
            k, v = (_decode64(s["pool"], s["table"], b, n, w) for w in (0, 1))
            first = n - c["Sq"]
        else:
            n = int(s["kv_lengths"][b]) if s["kv_lengths"] is not None else c["Sk"]
            k, v = (_hnd(s[x], lay)[b, :, :n].double() for x in ("k", "v"))
            first = c["Sk"] - c["Sq"]
        key = torch.arange(n, device=dev)
        rows = max(1, (1 << 26) // max(1, n))
        for h in range(c["hq"]):
            for a in range(0, c["Sq"], rows):
                e = min(c["Sq"], a + rows)
                pos = first + torch.arange(a, e, device=dev)[:, None]
                hidden = (key > pos) if c["causal"] else torch.zeros((e - a, n), dtype=torch.bool, device=dev)
                if c["window"]:
                    hidden = hidden | ((key <= pos - c["window"]) & (key >= c["sinks"]))
                z = (q[b, h, a:e] @ k[h // G].T * scale).masked_fill(hidden, -math.inf)
                w = torch.softmax(z, -1).masked_fill(hidden.all(-1, keepdim=True), 0.0)
                out[b, h, a:e] = w @ v[h // G]
    return _hnd(out, lay).contiguous()
