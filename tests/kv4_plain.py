"""Plain 64-bit forms of the 4-bit KV cache operators, written from the layout and the formulas."""
import math

import numpy as np
import torch

PAGE = 16


def places(D):
    """Byte and nibble of every (token, dim) of K and V in a page block, and bytes of the f16 scales."""
    G = D // 32
    t, d = np.arange(16)[:, None], np.arange(D)[None, :]
    g, r = d // 32, d % 32
    v0, pair = 8 * D + 64 * G, t // 2
    return {"k": (t * (D // 2) + (r // 8 * G + g) * 4 + r % 8 // 2, r % 2 + 0 * t), "ks": 8 * D + (t * G + g) * 2,
            "v": (v0 + ((pair * 8 + (r // 4 ^ 2 * (pair % 4))) * G + g) * 4 + t % 2 * 2 + r % 4 // 2, r % 2 + 0 * t),
            "vs": v0 + 8 * D + ((pair * G + g) * 2 + t % 2) * 2, "step": 32 * G}


def f16_at(block, at):
    return (block[..., at].astype(np.uint16) | block[..., at + 1].astype(np.uint16) << 8).view(np.float16).astype(np.float64)


def values(block, D):
    """K, V [.., 16, D] in 64 bits of page blocks [.., 20 D] (uint8)."""
    p, out = places(D), []
    for n in "kv":
        at, nib = p[n]
        c = (block[..., at] >> (4 * nib).astype(np.uint8)) & 15
        with np.errstate(invalid="ignore", over="ignore"):
            out.append(c * f16_at(block, p[n + "s"]) + f16_at(block, p[n + "s"] + p["step"]))
    return out


def quantized(x):
    """What x [.., D] (float64 of 16-bit inputs) reads back as."""
    y = np.clip(x, -65504, 65504).reshape(*x.shape[:-1], -1, 32)
    m = y.min(-1, keepdims=True).astype(np.float16).astype(np.float64)
    s = ((y.max(-1, keepdims=True) - m) / 15).astype(np.float16).astype(np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        c = np.where(s > 0, np.clip(np.rint((y - m) / np.where(s > 0, s, 1)), 0, 15), 0)
    return (c * s + m).reshape(x.shape), np.broadcast_to(s, y.shape).reshape(x.shape)


def attention(q, k, v, lens, scale=None, window=0, softcap=0.0, sinks=None):
    """q: list of [n_b, H, D]; k, v: lists of [ctx_b, Hkv, D]; all float64. The list of outputs, and for
    each the largest |v| its rows weigh."""
    outs = []
    for qb, kb, vb, c in zip(q, k, v, lens):
        n, H, D = qb.shape
        G = H // kb.shape[1] if kb.shape[1] else 1
        o = torch.zeros(n, H, D, dtype=torch.float64)
        for i in range(n):
            hi = c - n + i + 1
            lo = max(0, hi - window) if window > 0 else 0
            for h in range(H):
                if hi <= lo:
                    continue
                z = kb[lo:hi, h // G] @ qb[i, h] * (scale or 1 / math.sqrt(D))
                if softcap:
                    z = softcap * torch.tanh(z / softcap)
                top = z.max() if sinks is None else torch.maximum(z.max(), sinks[h])
                p = torch.exp(z - top)
                total = p.sum() + (0 if sinks is None else torch.exp(sinks[h] - top))
                o[i, h] = p @ vb[lo:hi, h // G] / total
        outs.append(o)
    return outs


def plan(old, new, table, free, head, cap):
    """Lists in, a dict of numpy int32 out; the table is changed."""
    slot, pos, seq = np.full(cap, -1, np.int32), np.zeros(cap, np.int32), np.full(cap, -1, np.int32)
    q_off, last, at = [0], [], 0
    for b, (o, n) in enumerate(zip(old, new)):
        have = -(-o // PAGE)
        for p in range(have, -(-(o + n) // PAGE)):
            table[b, p] = free[head]
            head += 1
        for p in range(o, o + n):
            slot[at], pos[at], seq[at] = table[b, p // PAGE] * PAGE + p % PAGE, p, b
            at += 1
        q_off.append(at)
        last.append(at - 1 if n else -1)
    return {"slot": slot, "pos": pos, "seq": seq, "q_off": np.array(q_off, np.int32),
            "ctx": np.array(old, np.int32) + np.array(new, np.int32), "last": np.array(last, np.int32),
            "free_head": np.array([head], np.int32)}
