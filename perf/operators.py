"""Operators of 4-bit KV serving, with their plain forms, as cases to be measured.

Four operators that one serving step chains:

* ``plan``      block tables, slot maps, positions and offsets of a ragged batch, from request lengths on the GPU;
* ``append``    K / V rows quantized into the pages of a 4-bit cache, read back as the values they stand for;
* ``attention`` single tokens (decode), a few tokens (verification) or chunks (prefill) over a 4-bit paged cache;
* ``logprobs``  log probability, rank, entropy and top alternatives of given tokens from logit rows.

4-bit page of one (page of 16 tokens, KV head), head dim D, groups of 32 dims (NG = D / 32), in bytes:

    K codes [16 tokens][4 t][NG groups] u32   dim = group * 32 + t * 8 + nibble (8 nibbles, lowest first)
    K scales [16][NG] f16, K minima [16][NG] f16
    V codes [8 token pairs][8 x][NG groups][2 tokens] u16   dim = group * 32 + g * 4 + nibble, g = x ^ 2 (pair % 4)
    V scales [8][NG][2] f16, V minima [8][NG][2] f16

A value is code * scale + minimum.  Quantization of a group x[32] (clamped to +-65504): minimum = f16(min x),
scale = f16((max x - minimum) / 15), code = rint((x - minimum) / scale) in [0, 15], 0 where the scale is 0.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda"
F16_MAX = 65504.0
DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's plan: 48 lanes advance by a token, three of them into a new page
        {"name": "plan decode 48", "op": "plan", "B": 48, "old_lo": 200, "old_hi": 9000, "new_lo": 1, "new_hi": 1},
        # admission of a burst of requests over cached prefixes (some fully cached: no new token)
        {"name": "plan ragged 333", "op": "plan", "B": 333, "old_lo": 0, "old_hi": 8192, "new_lo": 0, "new_hi": 256},
        # one decode step's K / V of 48 lanes, as slices of the fused q|k|v projection
        {"name": "append decode 48", "op": "append", "T": 48, "Hkv": 4, "D": 128, "dtype": "bf16", "fused": True},
        # a packed prefill chunk of several requests, an odd number of tokens
        {"name": "append chunk 8191", "op": "append", "T": 8191, "Hkv": 8, "D": 128, "dtype": "bf16", "fused": False},
        # one user, a short context: latency
        {"name": "decode 1x2048", "op": "attention", "B": 1, "lo": 2048, "hi": 2048, "n_lo": 1, "n_hi": 1, "H": 28, "Hkv": 4, "D": 128, "dtype": "bf16"},
        # five agents on about 9000 tokens each
        {"name": "decode 5x9000", "op": "attention", "B": 5, "lo": 8800, "hi": 9200, "n_lo": 1, "n_hi": 1, "H": 28, "Hkv": 4, "D": 128, "dtype": "bf16"},
        # a full serving batch with long, unequal contexts
        {"name": "decode 32x32k", "op": "attention", "B": 32, "lo": 7001, "hi": 32768, "n_lo": 1, "n_hi": 1, "H": 40, "Hkv": 8, "D": 128, "dtype": "bf16"},
        # verification of four drafted tokens plus one per lane, head dim 64
        {"name": "verify 16x5 D64", "op": "attention", "B": 16, "lo": 1003, "hi": 4097, "n_lo": 5, "n_hi": 5, "H": 64, "Hkv": 8, "D": 64, "dtype": "f16"},
        # the agents' turns: 256 new tokens each over a cached prefix
        {"name": "turn 5x256 over 8448", "op": "attention", "B": 5, "lo": 8448, "hi": 8704, "n_lo": 256, "n_hi": 256, "H": 28, "Hkv": 4, "D": 128, "dtype": "bf16"},
        # a long prompt's third chunk
        {"name": "chunk 4096 over 8192", "op": "attention", "B": 1, "lo": 12288, "hi": 12288, "n_lo": 4096, "n_hi": 4096, "H": 28, "Hkv": 4, "D": 128, "dtype": "bf16"},
        # log probabilities of a decode step's tokens
        {"name": "logprobs 5x152064", "op": "logprobs", "T": 5, "V": 152064, "k": 5, "dtype": "f32"},
        # scoring of a prompt: every position's token with 20 alternatives
        {"name": "logprobs 2048x152064", "op": "logprobs", "T": 2048, "V": 152064, "k": 20, "dtype": "f32"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))


def draw(rng):
    op = rng.choice(["plan", "append", "decode", "verify", "chunk", "logprobs"])
    if op == "plan":
        new = rng.choice([1, _log(rng, 2, 512)])
        return {"op": "plan", "B": _log(rng, 1, 512), "old_lo": 0, "old_hi": _log(rng, 16, 16384), "new_lo": 0 if new > 1 else 1, "new_hi": new}
    if op == "append":
        return {"op": "append", "T": _log(rng, 1, 8191), "Hkv": rng.choice([1, 2, 3, 4, 8]), "D": rng.choice([64, 128]),
                "dtype": rng.choice(["bf16", "f16"]), "fused": rng.random() < 0.5}
    if op == "logprobs":
        V = rng.choice([_log(rng, 500, 152064), 49152, 151936, 201088])
        return {"op": "logprobs", "T": min(_log(rng, 1, 2048), 311_000_000 // V), "V": V, "k": rng.choice([0, 1, 5, 20]), "dtype": rng.choice(["f32", "bf16"])}
    H, Hkv, D = rng.choice([(28, 4, 128), (40, 8, 128), (32, 4, 128), (9, 3, 64), (64, 8, 64), (8, 8, 64), (16, 1, 128), (7, 1, 128)])
    dt = rng.choice(["bf16", "f16"])
    if op == "chunk":
        n = _log(rng, 40, 2048)
        hi = n + _log(rng, 1, 8192)
        return {"op": "attention", "B": rng.randint(1, max(1, min(5, 2048 // n))), "lo": n + (hi - n) // 2, "hi": hi, "n_lo": n // 2, "n_hi": n,
                "H": H, "Hkv": Hkv, "D": D, "dtype": dt}
    n = 1 if op == "decode" else rng.randint(2, 9)
    hi = _log(rng, n, 32768)
    return {"op": "attention", "B": min(_log(rng, 1, 64), max(1, 400_000 // hi)), "lo": max(n, hi // rng.randint(1, 8)), "hi": hi, "n_lo": n, "n_hi": n,
            "H": H, "Hkv": Hkv, "D": D, "dtype": dt}


def _spread(lo, hi, B, by):
    """B whole numbers in [lo, hi], unequal, the same for every seed."""
    return [lo + int((hi - lo + 1) * ((0.37 + by * i) % 1.0)) for i in range(B)]


def _plan_lens(case):
    return (_spread(case["old_lo"], case["old_hi"], case["B"], 0.6180339887), _spread(case["new_lo"], case["new_hi"], case["B"], 0.7548776662))


def _attn_lens(case):
    """Context lengths (the new tokens among them) and new tokens."""
    return (_spread(case["lo"], case["hi"], case["B"], 0.6180339887), _spread(case["n_lo"], case["n_hi"], case["B"], 0.7548776662))


def page_bytes(D):
    return 16 * D + 4 * D


def work(case):
    if case["op"] == "plan":
        old, new = _plan_lens(case)
        opened = sum(-(-(a + n) // PAGE) - -(-a // PAGE) for a, n in zip(old, new))
        # lengths in; q_off, ctx, last out; per new token its page in, slot, position and request out; new pages in and into the table
        return {"bytes": 4.0 * (5 * case["B"] + 4 * sum(new) + 2 * opened), "flops": 0.0}
    if case["op"] == "append":
        rows = case["T"] * case["Hkv"]
        # K and V in, 4-bit rows out; read back: rows in, values out
        return {"bytes": rows * (2 * case["D"] * 2 + 2 * page_bytes(case["D"]) / PAGE + 2 * case["D"] * 2) + 8.0 * case["T"], "flops": 8.0 * rows * case["D"]}
    if case["op"] == "logprobs":
        return {"bytes": case["T"] * (case["V"] * (4.0 if case["dtype"] == "f32" else 2.0) + 16 + 8 * case["k"]), "flops": 6.0 * case["T"] * case["V"]}
    ctx, new = _attn_lens(case)
    pairs = sum(n * c - n * (n - 1) // 2 for c, n in zip(ctx, new))
    row = page_bytes(case["D"]) / PAGE
    return {"bytes": sum(ctx) * case["Hkv"] * row + 2 * 2.0 * sum(new) * case["H"] * case["D"], "flops": 4.0 * pairs * case["H"] * case["D"]}


# ------------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    return g


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _quant(x):
    """codes (uint8), scales and minima (f16) of x[..., D] in groups of 32."""
    x = x.float().clamp(-F16_MAX, F16_MAX)
    x = x.reshape(*x.shape[:-1], -1, 32)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    m = lo.half().float()
    s = ((hi - m) / torch.full_like(m, 15.0)).half().float()   # (a plain number would be multiplied by its reciprocal)
    code = torch.where(s > 0, torch.round((x - m) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(x)).clamp(0, 15)
    return code.to(torch.uint8), s.squeeze(-1).half(), m.squeeze(-1).half()


def _bytes(t):
    return t.contiguous().view(torch.uint8)


def _pairs():
    return torch.arange(8, device=DEV)[:, None]


def _crossed():
    """[pair, x]: which g stands at x (its own inverse)."""
    return torch.arange(8, device=DEV)[None, :] ^ (2 * (_pairs() % 4))


def _pack(k, v):
    """Pages [N, Hkv, bytes] of k, v [N, 16, Hkv, D]."""
    N, _, Hkv, D = k.shape
    G = D // 32
    kc, ks, km = _quant(k.transpose(1, 2))       # [N, Hkv, 16, G, 32], [N, Hkv, 16, G]
    kc = kc.reshape(N, Hkv, 16, G, 4, 4, 2)      # group, t, byte, nibble of the byte
    kc = (kc[..., 0] | (kc[..., 1] << 4)).transpose(3, 4)
    vc, vs, vm = _quant(v.transpose(1, 2))
    vc = vc.reshape(N, Hkv, 8, 2, G, 8, 2, 2)    # pair, token, group, g, byte, nibble
    vc = (vc[..., 0] | (vc[..., 1] << 4)).permute(0, 1, 2, 5, 4, 3, 6)   # pair, g, group, token, byte
    vc = vc[:, :, _pairs(), _crossed()]
    pairs = lambda t: t.reshape(N, Hkv, 8, 2, G).transpose(3, 4)  # noqa: E731
    parts = [kc, _bytes(ks), _bytes(km), vc, _bytes(pairs(vs)), _bytes(pairs(vm))]
    return torch.cat([p.reshape(N, Hkv, -1) for p in parts], dim=-1)


def _rows(g, shape, dtype):
    """Keys or values as a model makes them: normal, with offsets per channel and a few wide channels."""
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.bfloat16)
    D = shape[-1]
    off = torch.randn(D, generator=g, device=DEV) * 0.5
    wide = torch.where(torch.rand(D, generator=g, device=DEV) < 0.05, 4.0, 1.0)
    return (x * wide.to(x.dtype) + off.to(x.dtype)).to(dtype)


def prepare(case, seed):
    g = _gen(seed)
    if case["op"] == "plan":
        old, new = _plan_lens(case)
        B, T = case["B"], sum(new)
        width = max(1, max(-(-(a + n) // PAGE) for a, n in zip(old, new)))
        held = sum(-(-a // PAGE) for a in old)
        opened = sum(-(-(a + n) // PAGE) - -(-a // PAGE) for a, n in zip(old, new))
        ids = torch.randperm(held + opened + 64, generator=g, device=DEV).to(torch.int32) + 1
        n_old = torch.tensor([-(-a // PAGE) for a in old], device=DEV)
        at = torch.arange(width, device=DEV)[None, :]
        first = (torch.cumsum(n_old, 0) - n_old)[:, None]
        bt = torch.where(at < n_old[:, None], ids[(first + at).clamp(max=ids.numel() - 1)], torch.zeros_like(ids[:1]))
        return {"case": case, "old": _i32(old), "new": _i32(new), "table": bt.contiguous(), "free": ids[held:].contiguous(), "head": _i32([0]), "T": max(T, 1), "B": B}
    if case["op"] == "append":
        T, Hkv, D, dt = case["T"], case["Hkv"], case["D"], DT[case["dtype"]]
        if case["fused"]:   # k and v as slices of a projection's q|k|v rows
            qkv = _rows(g, (T, 4 * Hkv, D), dt)
            k, v = qkv[:, 2 * Hkv:3 * Hkv], qkv[:, 3 * Hkv:]
        else:
            k, v = _rows(g, (T, Hkv, D), dt), _rows(g, (T, Hkv, D), dt)
        P = -(-T // PAGE) + (T if T < 512 else 8)
        pages = torch.full((P, Hkv, page_bytes(D)), 255, dtype=torch.uint8, device=DEV)
        if T < 512:   # decode lanes: each in a page of its own
            slot = torch.randperm(P, generator=g, device=DEV)[:T] * PAGE + torch.randint(0, PAGE, (T,), generator=g, device=DEV)
        else:         # a chunk: runs of tokens over scattered pages
            page = torch.randperm(P, generator=g, device=DEV)
            at = torch.arange(T, device=DEV) + 5
            slot = page[at // PAGE] * PAGE + at % PAGE
        return {"case": case, "k": k, "v": v, "slot": slot.to(torch.int32), "pages": pages}
    if case["op"] == "logprobs":
        T, V, dt = case["T"], case["V"], DT[case["dtype"]]
        x = torch.randn((T, V), generator=g, device=DEV) * 2.5
        x += 6.0 * (torch.rand((T, V), generator=g, device=DEV) < 3.0 / V)        # a few likely tokens
        bad = torch.rand(V, generator=g, device=DEV) < 0.25
        x[::7] = torch.where(bad[None, :], torch.full_like(x[:1], -math.inf), x[::7])   # rows under a token mask
        tgt = torch.randint(0, V, (T,), generator=g, device=DEV)
        near = x.argmax(-1)
        tgt = torch.where(torch.rand(T, generator=g, device=DEV) < 0.6, near, tgt).to(torch.int32)
        if T > 8:
            tgt[3] = -1     # a position without a token to score
        return {"case": case, "x": x.to(dt), "target": tgt}
    ctx, new = _attn_lens(case)
    B, H, Hkv, D, dt = case["B"], case["H"], case["Hkv"], case["D"], DT[case["dtype"]]
    width = max(-(-c // PAGE) for c in ctx)
    n_pages = [-(-c // PAGE) for c in ctx]
    used = sum(n_pages)
    k = _rows(g, (used + 1, PAGE, Hkv, D), torch.bfloat16)
    v = _rows(g, (used + 1, PAGE, Hkv, D), torch.bfloat16)
    pages = _pack(k, v)
    ids = torch.randperm(used, generator=g, device=DEV).to(torch.int32) + 1
    np_ = torch.tensor(n_pages, device=DEV)
    at = torch.arange(width, device=DEV)[None, :]
    first = (torch.cumsum(np_, 0) - np_)[:, None]
    bt = torch.where(at < np_[:, None], ids[(first + at).clamp(max=used - 1)], torch.zeros_like(ids[:1])).contiguous()
    # page 0 belongs to nobody: its bytes are what memory held before (not-a-number scales)
    pages[0] = 255
    q = (torch.randn((sum(new), H, D), generator=g, device=DEV) * 1.5).to(dt)
    off = np.concatenate([[0], np.cumsum(new)])
    return {"case": case, "q": q, "pages": pages, "table": bt, "ctx": _i32(ctx), "q_off": _i32(off.tolist()), "max_new": max(new)}


# ------------------------------------------------------------------------------------- plain forms
def _unpack(pages, D):
    """K and V [.., 16, Hkv, D] in f32 of pages [.., Hkv, bytes]."""
    lead, Hkv, G = pages.shape[:-2], pages.shape[-2], D // 32
    sizes = [8 * D, 32 * G, 32 * G, 8 * D, 32 * G, 32 * G]
    kc, ks, km, vc, vs, vm = torch.split(pages, sizes, dim=-1)
    nib = lambda c: torch.stack([c & 15, c >> 4], -1)  # noqa: E731
    half = lambda c: c.contiguous().view(torch.float16).float()  # noqa: E731
    n = len(lead) + 1
    kc = nib(kc.reshape(*lead, Hkv, 16, 4, G, 4)).transpose(n + 1, n + 2).reshape(*lead, Hkv, 16, G, 32).float()
    k = kc * half(ks).reshape(*lead, Hkv, 16, G, 1) + half(km).reshape(*lead, Hkv, 16, G, 1)
    vc = nib(vc.reshape(-1, 8, 8, G, 2, 2)[:, _pairs(), _crossed()].reshape(*lead, Hkv, 8, 8, G, 2, 2))
    ax = list(range(n))                                         # then pair, g, group, token, byte, nibble
    vc = vc.permute(*ax, n, n + 3, n + 2, n + 1, n + 4, n + 5).reshape(*lead, Hkv, 16, G, 32).float()
    tok = lambda c: half(c).reshape(*lead, Hkv, 8, G, 2).transpose(-1, -2).reshape(*lead, Hkv, 16, G, 1)  # noqa: E731
    v = vc * tok(vs) + tok(vm)
    shape = (*lead, Hkv, 16, D)
    return k.reshape(shape).transpose(-2, -3), v.reshape(shape).transpose(-2, -3)


def _plain_plan(s):
    old, new, table, free = s["old"].long(), s["new"].long(), s["table"].clone(), s["free"]
    B, W, T = s["B"], table.shape[1], s["T"]
    have, need = (old + PAGE - 1) // PAGE, (old + new + PAGE - 1) // PAGE
    opened = need - have
    base = torch.cumsum(opened, 0) - opened + s["head"].long()
    at = torch.arange(W, device=DEV)[None, :]
    fresh = (at >= have[:, None]) & (at < need[:, None])
    table = torch.where(fresh, free[(base[:, None] + at - have[:, None]).clamp(0, free.numel() - 1)], table)
    q_off = torch.cat([torch.zeros_like(new[:1]), torch.cumsum(new, 0)])
    i = torch.arange(T, device=DEV)
    seq = (i[:, None] >= q_off[None, 1:]).sum(1)
    live = i < q_off[-1]
    sq = seq.clamp(max=B - 1)
    pos = torch.where(live, old[sq] + i - q_off[sq], torch.zeros_like(i))
    slot = torch.where(live, table[sq, pos // PAGE].long() * PAGE + pos % PAGE, torch.full_like(i, -1))
    last = torch.where(new > 0, q_off[1:] - 1, torch.full_like(new, -1))
    out = {"slot": slot, "pos": pos, "seq": torch.where(live, seq, torch.full_like(seq, -1)), "q_off": q_off, "ctx": old + new, "last": last,
           "head": s["head"].long() + opened.sum()}
    return {**{n: t.to(torch.int32) for n, t in out.items()}, "table": table}


def _plain_append(s):
    D = s["case"]["D"]
    back = []
    for x in (s["k"], s["v"]):
        c, sc, m = _quant(x)
        y = c.float() * sc.float()[..., None] + m.float()[..., None]
        back.append(y.reshape(*x.shape[:-1], D).to(torch.bfloat16))
    return back


def _plain_attention(s):
    case = s["case"]
    B, H, Hkv, D = case["B"], case["H"], case["Hkv"], case["D"]
    N, W = s["max_new"], s["table"].shape[1]
    k, v = _unpack(s["pages"][s["table"].long()], D)             # [B, W, 16, Hkv, D]
    ctx, q_off = s["ctx"].long(), s["q_off"].long()
    new = q_off[1:] - q_off[:-1]
    at = torch.arange(W * PAGE, device=DEV)
    there = (at[None, :] < ctx[:, None])[..., None, None]
    zero = torch.zeros((), device=DEV)
    k = torch.where(there, k.reshape(B, W * PAGE, Hkv, D), zero).permute(0, 2, 3, 1)
    v = torch.where(there, v.reshape(B, W * PAGE, Hkv, D), zero).transpose(1, 2)
    i = torch.arange(N, device=DEV)
    row = (q_off[:-1, None] + i[None, :]).clamp(max=s["q"].shape[0] - 1)
    q = s["q"].float()[row].reshape(B, N, Hkv, H // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = torch.matmul(q, k).reshape(B, Hkv, H // Hkv, N, W * PAGE) / math.sqrt(D)
    pos = ctx[:, None] - new[:, None] + i[None, :]
    seen = (at[None, None, :] <= pos[..., None])[:, None, None]
    x = torch.where(seen, x, torch.full((), -math.inf, device=DEV))
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = torch.matmul(x.reshape(B, Hkv, -1, W * PAGE), v).reshape(B, Hkv, H // Hkv, N, D).permute(0, 3, 1, 2, 4).reshape(B, N, H, D)
    live = i[None, :] < new[:, None]
    return o[live].to(s["q"].dtype)


def _plain_logprobs(s):
    case = s["case"]
    T, V, k = case["T"], case["V"], case["k"]
    x = s["x"].float()
    t = s["target"].long()
    given = (t >= 0) & (t < V)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e > 0, e * (x - top), torch.zeros((), device=DEV)).sum(-1, keepdim=True) / total)[:, 0]
    xt = x.gather(1, t.clamp(0, V - 1)[:, None])
    lp = torch.where(given, (xt - top - log_total)[:, 0], torch.zeros((), device=DEV))
    i = torch.arange(V, device=DEV)[None, :]
    rank = torch.where(given, 1 + ((x > xt) | ((x == xt) & (i < t[:, None]))).sum(-1), torch.zeros_like(t))
    out = {"logprob": lp, "entropy": entropy, "rank": rank.to(torch.int32)}
    if k:
        b = (x + 0.0).view(torch.int32)
        key = torch.where(b >= 0, b, b ^ 0x7FFFFFFF).long() * (1 << 32) + (0xFFFFFFFF - i)   # ties go to the lowest index
        ids = 0xFFFFFFFF - (torch.topk(key, k, dim=-1).values & 0xFFFFFFFF)
        out["top_ids"] = ids.to(torch.int32)
        out["top_logprobs"] = x.gather(1, ids) - top - log_total
    return out


# ------------------------------------------------------------------------------------- one pass
def run(state):
    op = state["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[op](state)
    from fak_b200.ops import kernels as K
    if op == "plan":
        p = K.plan_batch(state["old"], state["new"], state["table"], state["free"], state["head"], state["T"])
        return {"slot": p.slot, "pos": p.pos, "seq": p.seq, "q_off": p.q_off, "ctx": p.ctx, "last": p.last, "head": p.free_head, "table": state["table"]}
    if op == "append":
        K.kv4_append(state["k"], state["v"], state["slot"], state["pages"])
        return list(K.kv4_read(state["pages"], state["slot"], state["case"]["D"], torch.bfloat16))
    if op == "logprobs":
        r = K.token_logprobs(state["x"], state["case"]["V"], state["target"], state["case"]["k"])
        out = {"logprob": r.logprob, "entropy": r.entropy, "rank": r.rank}
        return {**out, "top_ids": r.top_ids, "top_logprobs": r.top_logprobs} if state["case"]["k"] else out
    q = state["q"]
    out = torch.empty_like(q)
    if state["max_new"] == 1:
        K.kv4_decode_attention(q, state["pages"], state["table"], state["ctx"], out)
    else:
        K.kv4_prefill_attention(q, state["pages"], state["table"], state["q_off"], state["ctx"], out, state["max_new"])
    return out


# ------------------------------------------------------------------------------------- 64 bits
def _read64(page, D):
    """K, V [16, D] of one (page, head)'s bytes (numpy uint8 [.., bytes] -> [.., 16, D]), value by value from the layout."""
    G = D // 32
    d, t = np.arange(D), np.arange(16)
    grp, r = d // 32, d % 32
    k_at = t[:, None] * (D // 2) + ((r // 8) * G + grp) * 4 + (r % 8) // 2
    v0 = 8 * D + 64 * G
    pair = t[:, None] // 2
    v_at = v0 + ((pair * 8 + ((r // 4) ^ (2 * (pair % 4)))) * G + grp) * 4 + (t[:, None] % 2) * 2 + (r % 4) // 2
    ks_at = 8 * D + (t[:, None] * G + grp) * 2
    vs_at = v0 + 8 * D + (((t[:, None] // 2) * G + grp) * 2 + t[:, None] % 2) * 2

    def f16(at):
        return (page[..., at].astype(np.uint16) | (page[..., at + 1].astype(np.uint16) << 8)).view(np.float16).astype(np.float64)

    k = ((page[..., k_at] >> (4 * (r % 2))) & 15).astype(np.float64) * f16(ks_at) + f16(ks_at + 32 * G)
    v = ((page[..., v_at] >> (4 * (r % 2))) & 15).astype(np.float64) * f16(vs_at) + f16(vs_at + 32 * G)
    return k, v


def exact(case, seed):
    if case["op"] == "plan":
        return None      # whole numbers only
    if case["op"] == "attention" and work(case)["bytes"] > 3e8:
        return None
    s = prepare(case, seed)
    if case["op"] == "append":
        out = []
        for x in (s["k"], s["v"]):
            x = x.double().cpu().numpy()
            x = x.reshape(*x.shape[:-1], -1, 32)
            m = x.min(-1, keepdims=True).astype(np.float16).astype(np.float64)
            sc = ((x.max(-1, keepdims=True) - m) / 15).astype(np.float16).astype(np.float64)
            c = np.clip(np.rint((x - m) / np.where(sc > 0, sc, 1.0)), 0, 15) * (sc > 0)
            out.append(torch.from_numpy((c * sc + m).reshape(case["T"], case["Hkv"], case["D"])))
        return out
    if case["op"] == "logprobs":
        T, V, k = case["T"], case["V"], case["k"]
        lp, ent, tops = [], [], []
        for r in range(T):
            x = s["x"][r].double()
            z = torch.log_softmax(x, 0)
            p = torch.exp(z)
            t = int(s["target"][r])
            lp.append(float(z[t]) if 0 <= t < V else 0.0)
            ent.append(-(p * torch.where(p > 0, z, torch.zeros_like(z))).sum())
            if k:
                tops.append(torch.sort(z, descending=True).values[:k] if T <= 64 else torch.topk(z, k).values)
        out = {"logprob": torch.tensor(lp, dtype=torch.float64), "entropy": torch.stack(ent), "rank": None}
        return {**out, "top_ids": None, "top_logprobs": torch.stack(tops)} if k else out
    ctx, new = _attn_lens(case)
    H, Hkv, D = case["H"], case["Hkv"], case["D"]
    out, at = [], 0
    pages, table = s["pages"].cpu().numpy(), s["table"].cpu().numpy()
    for b, (c, n) in enumerate(zip(ctx, new)):
        page = pages[table[b, :-(-c // PAGE)]]
        k, v = (torch.from_numpy(a.transpose(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :c].copy()).to(DEV) for a in _read64(page, D))
        q = s["q"][at:at + n].double().reshape(n, Hkv, H // Hkv, D)
        at += n
        hide = torch.arange(c, device=DEV)[None, :] > torch.arange(c - n, c, device=DEV)[:, None]
        heads = []
        for h in range(H):
            z = q[:, h // (H // Hkv), h % (H // Hkv)] @ k[h // (H // Hkv)].T / math.sqrt(D)
            heads.append(torch.softmax(z.masked_fill(hide, -math.inf), -1) @ v[h // (H // Hkv)])
        out.append(torch.stack(heads, 1))
    return torch.cat(out)
