"""Chunks and few rows over the 4-bit cache in every form: both kernels, types, windows, soft-caps, sinks, splits, strides.

With u = 2^-11, f16's unit roundoff (a uniform rounding error has the standard deviation u / sqrt 3):
* a logit carries the roundings of the dequantized keys (tiles) and of f32 queries, independent ones, so its
  standard deviation is at most a = scale sqrt(sum q_d^2 k_d^2) u / sqrt 3, twice that in variance where both round;
* tiles round a probability and a value once each: the relative error of a term is sqrt(a^2 + 2 u^2 / 3);
* rows round a probability and its product with a scale; the product meets a code, up to 2.5 times the value's
  size (c s = v - m, m the group's minimum): sqrt(a^2 + u^2 / 3 + (2.5 u)^2 / 3).
Every output lies within six of these of the largest value, twice for what numerator and denominator share;
their root mean square within two of the outputs' own.  Rounding the output comes on top."""
import math

import numpy as np
import pytest
import torch

import kv4_plain as plain
from test_kv4_edges_gpu import OUT_U, U16, cache, dev, gen

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def term(q, k, scale, dtype, tiles):
    """Standard deviation of a term's relative error (the largest over rows of q [n, H, D] and keys k [c, Hkv, D])."""
    G = q.shape[1] // k.shape[1]
    a2 = torch.einsum("nhgd,chd->nhgc", q.reshape(q.shape[0], -1, G, q.shape[2]) ** 2, k ** 2).max().item() * scale ** 2 * U16 ** 2 / 3
    a2 *= (1 if tiles else 0) + (1 if dtype == torch.float32 else 0)
    return math.sqrt(a2 + 2 * U16 ** 2 / 3) if tiles else math.sqrt(a2 + U16 ** 2 / 3 + (2.5 * U16) ** 2 / 3)


def check(out, want, vs, sigma):
    out, u = out.double().cpu(), OUT_U[out.dtype]
    err = (out - want).abs()
    assert (err <= 12 * sigma * vs.abs().max() + u * want.abs()).all()
    assert err.pow(2).mean().sqrt() <= 2 * math.sqrt(sigma ** 2 + u ** 2 / 3) * want.pow(2).mean().sqrt()


def rows(g, shape):
    return torch.randn(shape, generator=g, device="cuda") + 0.5 * torch.randn(shape[-1], generator=g, device="cuda")


CASES = [  # cached, new, H, Hkv, D
    ([1100, 0, 30], [9, 40, 0], 8, 2, 128), ([700], [37], 7, 1, 64), ([2100, 900], [3, 5], 16, 4, 64), ([5, 300], [150, 20], 2, 2, 128),
]
FORMS = [{}, {"window": 200}, {"softcap": 15.0}, {"sinks": True}, {"window": 333, "softcap": 8.0, "sinks": True, "scale": 0.2}]


@pytest.mark.parametrize("old,new,H,Hkv,D", CASES)
@pytest.mark.parametrize("form", FORMS, ids=lambda f: "+".join(f) or "plain")
def test_forms(K, old, new, H, Hkv, D, form):
    lens, T, g = [a + n for a, n in zip(old, new)], sum(new), gen(sum(new) + D)
    pages, table, ks, vs = cache(K, [rows(g, (c, Hkv, D)) for c in lens], [rows(g, (c, Hkv, D)) for c in lens])
    form = dict(form)
    sinks = torch.randn(H, generator=g, device="cuda") * 2 + 3 if form.pop("sinks", False) else None
    scale = form.get("scale", 1 / math.sqrt(D))
    off = np.concatenate([[0], np.cumsum(new)])
    base = torch.randn(T, H, D, generator=g, device="cuda") * 1.3
    for dtype in (torch.float32, torch.float16, torch.bfloat16):
        q = base.to(dtype)
        qs = [q[off[b]:off[b + 1]].double().cpu() for b in range(len(new))]
        want = plain.attention(qs, ks, vs, lens, sinks=None if sinks is None else sinks.double().cpu(), **form)
        for tiles in (False, True):
            for n_split in (0, 1, 3, 6):
                out = torch.full((T + 1, H, D), 7, dtype=dtype, device="cuda")
                K.kv4_prefill_attention(q, pages, table, dev(off), dev(lens), out[:T], max(new), sinks=sinks, n_split=n_split,
                                        tiles=tiles, **form)
                for b in range(len(new)):
                    if new[b]:
                        check(out[off[b]:off[b + 1]], want[b], vs[b], term(qs[b], ks[b], scale, dtype, tiles))
                assert (out[T] == 7).all()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("by", [1, 4, 8])
def test_strides(K, tiles, dtype, by):
    """Rows of q and out ``by`` elements off vector boundaries, in offset, heads and tokens: the same bits."""
    lens, n, H, D, g = [400], 150, 4, 64, gen(by)
    pages, table, ks, vs = cache(K, [rows(g, (400, 2, D))], [rows(g, (400, 2, D))])
    q = torch.randn(n, H, D, generator=g, device="cuda").to(dtype)
    want = torch.empty_like(q)
    K.kv4_prefill_attention(q, pages, table, dev([0, n]), dev(lens), want, n, tiles=tiles)
    for shape, cut in (((n * H * D + by,), lambda b: b[by:].view(n, H, D)), ((n, H, D + by), lambda b: b[:, :, :D]),
                       ((n, H * D + by), lambda b: b[:, :H * D].view(n, H, D)), ((H, n, D), lambda b: b.transpose(0, 1))):
        qb, ob = torch.zeros(shape, dtype=dtype, device="cuda"), torch.full(shape, 7, dtype=dtype, device="cuda")
        cut(qb).copy_(q)
        for x, o in ((cut(qb), want.clone()), (q, cut(ob)), (cut(qb), cut(ob))):
            K.kv4_prefill_attention(x, pages, table, dev([0, n]), dev(lens), o, n, tiles=tiles)
            assert torch.equal(o, want)
        cut(ob).fill_(7)
        assert (ob == 7).all()


@pytest.mark.parametrize("tiles", [False, True])
def test_types_of_their_own(K, tiles):
    """q and out may differ in type."""
    lens, n, H, D, g = [300], 90, 4, 128, gen(5)
    pages, table, ks, vs = cache(K, [rows(g, (300, 1, D))], [rows(g, (300, 1, D))])
    q = torch.randn(n, H, D, generator=g, device="cuda").to(torch.bfloat16)
    want = plain.attention([q.double().cpu()], ks, vs, lens)[0]
    for x in (q, q.float()):
        for dtype in (torch.float32, torch.float16, torch.bfloat16):
            out = torch.empty(n, H, D, dtype=dtype, device="cuda")
            K.kv4_prefill_attention(x, pages, table, dev([0, n]), dev(lens), out, n, tiles=tiles)
            check(out, want, vs[0], term(q.double().cpu(), ks[0], D ** -0.5, torch.bfloat16, tiles))


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("n_split", [0, 4])
def test_calls_repeat_their_bits(K, tiles, n_split):
    lens, new, H, D, g = [900, 333, 64], [70, 33, 64], 14, 128, gen(6)
    pages, table, ks, vs = cache(K, *([rows(g, (c, 2, D)) for c in lens] for _ in "kv"))
    q = torch.randn(sum(new), H, D, generator=g, device="cuda")
    off = dev(np.concatenate([[0], np.cumsum(new)]))
    outs = [torch.empty_like(q) for _ in range(12)]
    for o in outs:
        K.kv4_prefill_attention(q, pages, table, off, dev(lens), o, max(new), tiles=tiles, n_split=n_split)
    assert all(torch.equal(o, outs[0]) for o in outs)


@pytest.mark.parametrize("tiles", [False, True])
def test_sequences_with_less_context_than_new_tokens(K, tiles):
    """Rows before the first key see nothing: zeros, sinks or not; the others see theirs."""
    lens, new, H, D, g = [5, 0, 33], [9, 4, 40], 4, 64, gen(8)
    pages, table, ks, vs = cache(K, *([rows(g, (c, 2, D)) for c in lens] for _ in "kv"))
    q = torch.randn(sum(new), H, D, generator=g, device="cuda").half()
    off = np.concatenate([[0], np.cumsum(new)])
    for sinks in (None, torch.zeros(H, device="cuda")):
        want = plain.attention([q[off[b]:off[b + 1]].double().cpu() for b in range(3)], ks, vs, lens,
                               sinks=None if sinks is None else sinks.double().cpu())
        out = torch.full_like(q, 7)
        K.kv4_prefill_attention(q, pages, table, dev(off), dev(lens), out, max(new), tiles=tiles, sinks=sinks)
        assert (out[:4] == 0).all() and (out[9:13] == 0).all() and (out[13:20] == 0).all()
        for b in (0, 2):
            check(out[off[b]:off[b + 1]], want[b], vs[b], term(q.double().cpu(), ks[b], D ** -0.5, torch.float16, tiles))


@pytest.mark.parametrize("old,new,H,Hkv,D", [([1700], [300], 1, 1, 64), ([900, 3], [100, 130], 4, 2, 128), ([40, 700], [9, 5], 8, 1, 64),
                                             ([0], [20], 2, 2, 128), ([2500], [260], 2, 1, 64)])
@pytest.mark.parametrize("window", [0, 150, 700])
@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("deep", [True, False])
def test_values_that_are_no_numbers_reach_the_rows_that_see_them(K, old, new, H, Hkv, D, window, tiles, deep):
    """NaN values in one or all groups of some tokens, among the keys that all rows see, some, or none: a row's group
    is NaN exactly where it sees one, and everything else is as if they were 0."""
    lens, g = [a + n for a, n in zip(old, new)], gen(sum(new) + window)
    kr, vr, bad = [], [], []
    for a, c in zip(old, lens):
        kr.append(rows(g, (c, Hkv, D)))
        v = rows(g, (c, Hkv, D))
        at = sorted({c // 3, max(0, a - 200), max(0, a - 60), max(0, a - 1), min(c - 1, a + 2), (a + c) // 2, c - 1})
        at = at if deep else [j for j in at if j > a]      # (without a window, every row sees those before)
        b = torch.zeros(c, Hkv, D // 32, dtype=torch.bool)
        for i, j in enumerate(at):
            b[j, i % Hkv, slice(None) if i % 3 == 0 else slice(i % (D // 32), i % (D // 32) + 1)] = True
        v.view(c, Hkv, D // 32, 32)[b.cuda()] = math.nan
        vr.append(v)
        bad.append(b)
    pages, table, ks, vs = cache(K, kr, vr)
    assert all(torch.equal(torch.isnan(v.view(*b.shape, 32)), b[..., None].expand(*b.shape, 32)) for v, b in zip(vs, bad))
    vs = [torch.nan_to_num(v, nan=0.0) for v in vs]
    off = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(sum(new), H, D, generator=g, device="cuda").half()
    qs = [q[off[b]:off[b + 1]].double().cpu() for b in range(len(new))]
    want = plain.attention(qs, ks, vs, lens, window=window)
    for n_split in (1, 3, 0, 20):
        out = torch.empty_like(q)
        K.kv4_prefill_attention(q, pages, table, dev(off), dev(lens), out, max(new), window=window, tiles=tiles, n_split=n_split)
        for b, (c, n) in enumerate(zip(lens, new)):
            hi = torch.arange(c - n + 1, c + 1)[:, None]
            j = torch.arange(c)[None, :]
            sees = ((j < hi) & (j >= (hi - window if window else 0))).double()                    # [n, c]
            hit = torch.einsum("nc,chg->nhg", sees, bad[b].double()) > 0                          # [n, Hkv, groups]
            hit = hit.repeat_interleave(H // Hkv, 1).repeat_interleave(32, 2)
            o = out[off[b]:off[b + 1]]
            assert torch.equal(torch.isnan(o).cpu(), hit)
            if not hit.all():
                check(o[~hit.cuda()], want[b][~hit], vs[b], term(qs[b], ks[b], D ** -0.5, torch.float16, tiles))


@pytest.mark.parametrize("old,new,H,Hkv,D", [([700], [300], 1, 1, 64), ([100, 9], [60, 130], 4, 2, 128), ([40, 300], [9, 5], 8, 1, 64)])
@pytest.mark.parametrize("window", [0, 150])
@pytest.mark.parametrize("tiles", [False, True])
def test_keys_and_queries_that_are_no_numbers_stay_with_their_rows(K, old, new, H, Hkv, D, window, tiles):
    lens, g = [a + n for a, n in zip(old, new)], gen(sum(new) + window)
    kr, vr, bad = [], [], []
    for a, c in zip(old, lens):
        k = rows(g, (c, Hkv, D))
        b = torch.zeros(c, Hkv, dtype=torch.bool)
        b[min(c - 1, a + 3), 0] = b[(a + c) // 2, -1] = True
        k[b.cuda()] = math.nan
        kr.append(k)
        vr.append(rows(g, (c, Hkv, D)))
        bad.append(b)
    pages, table, ks, vs = cache(K, kr, vr)
    ks = [torch.nan_to_num(k, nan=0.0) for k in ks]
    off = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(sum(new), H, D, generator=g, device="cuda").half()
    broken = torch.zeros(sum(new), H, dtype=torch.bool)
    broken[1, 0] = broken[-1, -1] = True
    want = plain.attention([q[off[b]:off[b + 1]].double().cpu() for b in range(len(new))], ks, vs, lens, window=window)
    sigma = [term(q[off[b]:off[b + 1]].double().cpu(), ks[b], D ** -0.5, torch.float16, tiles) for b in range(len(new))]
    q[1, 0, 5], q[-1, -1, 0] = math.nan, math.nan
    for n_split in (1, 3, 0, 20):
        out = torch.empty_like(q)
        K.kv4_prefill_attention(q, pages, table, dev(off), dev(lens), out, max(new), window=window, tiles=tiles, n_split=n_split)
        for b, (c, n) in enumerate(zip(lens, new)):
            hi = torch.arange(c - n + 1, c + 1)[:, None]
            j = torch.arange(c)[None, :]
            sees = ((j < hi) & (j >= (hi - window if window else 0))).double()
            hit = (torch.einsum("nc,ch->nh", sees, bad[b].double()) > 0).repeat_interleave(H // Hkv, 1) | broken[off[b]:off[b + 1]]
            o = out[off[b]:off[b + 1]]
            assert torch.equal(torch.isnan(o).cpu(), hit[..., None].expand(n, H, D))
            check(o[~hit.cuda()], want[b][~hit], vs[b], sigma[b])
