"""Generation in chunks over a rolling 4-bit cache, on synthetic activations.

Shows the cache and window operators as a generator uses them: the prompt
attends through ``ops.window_attention`` while its K/V go into a ``KV4Cache``;
every later chunk (a video chunk, drafted tokens, one token) is rotated,
quantised and appended by one call and attends over the cache by another; pages
behind the window return to the pool.  Each chunk's output is compared with
exact attention in FP32 over the unquantised tokens (what the 4 bits cost) and
timed with CUDA events.

    python -m vc_attention.streaming [--prompt 2048] [--chunks 256,16,1,1] [--window 1024] [--sinks 16]
"""
from __future__ import annotations

import argparse
import json

import torch

from vc_b200 import ops
from vc_b200.kv_cache import KV4Cache


def rotation(head_dim: int, positions: int, device, base: float = 10000.0):
    """FP32 cos and sin [positions, head_dim/2] of half-style rotation."""
    freq = base ** (-torch.arange(0, head_dim, 2, device=device, dtype=torch.float64) / head_dim)
    angle = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def rotate(x, cos, sin):
    """Half-style rotation of [B,H,S,D] by rows of cos and sin [S,D/2], in FP32."""
    a, b = x.float().chunk(2, -1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def exact(q, k, v, first, window, sinks):
    """FP32 attention of queries at positions first.. over all tokens; HND, shared heads repeated."""
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = q @ k.transpose(-1, -2) * q.shape[-1] ** -0.5
    i = first + torch.arange(q.shape[2], device=q.device)[:, None]
    j = torch.arange(k.shape[2], device=q.device)[None, :]
    ok = (j <= i) & ((j > i - window) | (j < sinks))
    return torch.softmax(s.masked_fill(~ok, float("-inf")), -1) @ v


@torch.no_grad()
def run(prompt=2048, chunks=(256, 16, 1, 1), *, batch=1, heads=28, kv_heads=4, head_dim=128, window=1024, sinks=16,
        page_size=64, dtype=torch.bfloat16, seed=0, device="cuda"):
    """One report per stage: tokens, milliseconds, relative error against exact attention, free pages."""
    total = prompt + sum(chunks)
    g = torch.Generator(device=device).manual_seed(seed)
    draw = lambda h: torch.randn((batch, h, total, head_dim), generator=g, device=device).to(dtype)
    q, k, v = draw(heads), draw(kv_heads), draw(kv_heads)
    cos, sin = rotation(head_dim, total, device)
    rq, rk, fv = rotate(q, cos, sin), rotate(k, cos, sin), v.float()
    cache = KV4Cache(batch, kv_heads, head_dim, pages=batch * -(-total // page_size), max_tokens=total,
                     page_size=page_size, cos=cos, sin=sin, window=window, sinks=sinks, device=device)
    reports, at = [], 0
    for n in (prompt, *chunks):
        part = slice(at, at + n)
        t0, t1 = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        t0.record()
        turned = cache.append(k[:, :, part], v[:, :, part], q[:, :, part])
        if at == 0:   # the prompt has its K/V at hand in 16 bits
            out = ops.window_attention(turned, rk[:, :, part].to(dtype), v[:, :, part], window=window, sinks=sinks)
        else:
            out = cache.attend(turned)
        t1.record()
        freed = cache.trim()
        want = exact(rq[:, :, part], rk[:, :, :at + n], fv[:, :, :at + n], at, window, sinks)
        t1.synchronize()
        reports.append({"tokens": n, "ms": t0.elapsed_time(t1), "pages_freed": freed, "pages_free": cache.free_pages,
                        "rel_l2": float((out.float() - want).norm() / want.norm())})
        at += n
    return reports


def main():
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--prompt", type=int, default=2048)
    ap.add_argument("--chunks", default="256,16,1,1")
    ap.add_argument("--window", type=int, default=1024)
    ap.add_argument("--sinks", type=int, default=16)
    a = ap.parse_args()
    for r in run(a.prompt, tuple(int(x) for x in a.chunks.split(",")), window=a.window, sinks=a.sinks):
        print(json.dumps(r))


if __name__ == "__main__":
    main()
