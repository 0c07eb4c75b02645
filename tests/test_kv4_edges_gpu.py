"""4-bit KV cache on the GPU where it can go wrong: rows between vector boundaries, values of every size, masks,
argument ranges."""
import math

import numpy as np
import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def dev(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("odd", ["offset", "head stride", "row stride", "page stride", "v only"])
@pytest.mark.parametrize("by", [1, 2, 4])
def test_append_rows_between_vector_boundaries(K, D, dtype, odd, by):
    """Rows that start ``by`` elements past a 16-byte boundary (4 16-bit elements are 8 bytes), through each of
    the offset and the strides of token rows and of 16-bit cache pages: the formula's values, exactly."""
    T, Hkv, P = 37, 3, 4
    g = gen(D + by)
    x = torch.randn(2, 64, Hkv, D, generator=g, device="cuda").to(torch.bfloat16).to(dtype)   # (the same codes in 32 and 64 bits)
    x[1] += 0.25

    def place(x, odd):
        if odd == "page stride":       # pages [P, Hkv, 16, D] with ``by`` elements between them
            buf = torch.zeros(P, Hkv * 16 * D + by, dtype=dtype, device="cuda")
            y = buf[:, :Hkv * 16 * D].view(P, Hkv, 16, D)
            return y.copy_(x.view(P, 16, Hkv, D).transpose(1, 2))
        if odd == "head stride":
            y = torch.zeros(T, Hkv, D + by, dtype=dtype, device="cuda")[:, :, :D]
        elif odd == "row stride":
            y = torch.zeros(T, Hkv * D + by, dtype=dtype, device="cuda")[:, :Hkv * D].view(T, Hkv, D)
        else:
            y = torch.zeros(T * Hkv * D + by, dtype=dtype, device="cuda")[by if odd == "offset" else 0:][:T * Hkv * D].view(T, Hkv, D)
        return y.copy_(x[:T])

    k, v = place(x[0], "" if odd == "v only" else odd), place(x[1], "offset" if odd == "v only" else odd)
    slot = torch.randperm(P * 16, generator=g, device="cuda")[:T].to(torch.int32)
    pages = torch.full((P, Hkv, K.kv4_page_bytes(D)), 255, dtype=torch.uint8, device="cuda")
    K.kv4_append(k, v, slot, pages)
    for got, src in zip(K.kv4_read(pages, slot, D, torch.float32), x):
        want, _ = plain.quantized(src[:T].double().cpu().numpy())
        np.testing.assert_array_equal(got.double().cpu().numpy(), want.astype(np.float32).astype(np.float64))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_append_of_the_widest_groups(K, D, dtype):
    """-65504 + 15 f16(131008 / 15) is 65536, past f16: the scale is one step less, 8728, and the largest value 65416.
    Attention rounds values to f16, so it has to stay finite."""
    x = torch.linspace(-65504, 65504, 32, device="cuda").repeat(D // 32).view(1, 1, D).to(dtype)
    pages = torch.zeros(1, 1, K.kv4_page_bytes(D), dtype=torch.uint8, device="cuda")
    K.kv4_append(x, x, dev([0]), pages)
    want = torch.round((x.double() + 65504) / 8728).clamp(0, 15) * 8728 - 65504
    for r in K.kv4_read(pages, dev([0]), D, torch.float32):
        assert torch.equal(r.double(), want) and r.max() == 65416
    q = torch.zeros(1, 1, D, device="cuda")
    for tiles in (False, True):
        out = torch.empty_like(q)
        K.kv4_prefill_attention(q, pages, dev([[0]]), dev([0, 1]), dev([1]), out, 1, tiles=tiles)
        assert ((out.double() - want).abs() <= 4 * U16 * 65504).all()


# ------------------------------------------------------------------------------------ attention
U16 = 2.0 ** -11
OUT_U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def cache(K, ks, vs):
    """A cache of the rows ks, vs (lists of [c, Hkv, D]): pages, table, and the values it stands for (64 bits)."""
    n = [max(1, -(-k.shape[0] // 16)) for k in ks]
    Hkv, D = ks[0].shape[1:]
    pages = torch.full((sum(n) + 1, Hkv, K.kv4_page_bytes(D)), 255, dtype=torch.uint8, device="cuda")   # NaN scales
    table = torch.zeros(len(ks), max(n), dtype=torch.int32, device="cuda")
    at, rk, rv = 1, [], []
    for b, (k, v) in enumerate(zip(ks, vs)):
        table[b, :n[b]] = torch.arange(at, at + n[b], device="cuda").flip(0)
        at += n[b]
        j = torch.arange(k.shape[0], device="cuda")
        slot = (table[b, j // 16] * 16 + j % 16).to(torch.int32)
        K.kv4_append(k, v, slot, pages)
        for out, r in zip((rk, rv), K.kv4_read(pages, slot, D, torch.float32)):
            out.append(r.double().cpu())
    return pages, table, rk, rv


def product_step(c):
    """What the products of probabilities and scales may lose to f16's smallest step, over c keys: half a step
    each, times the largest code, against a sum that holds a probability of 2^15 (scales below 1)."""
    return c * 15 * 2.0 ** -25 / 2.0 ** 15


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-5])
@pytest.mark.parametrize("logit", [0.0, 7.0, 10.0])
def test_small_values_under_a_key_that_stands_out(K, D, size, logit):
    """One key's logit lies ``logit`` above thousands of equal ones, values of every magnitude: the others' share
    must survive their products with small scales.  Tolerance as for decode (4 roundings of the largest value),
    plus f16's smallest step."""
    c, H = 4000, 3
    g = gen(7)
    k, v = torch.randn(c, 1, D, generator=g, device="cuda"), torch.randn(c, 1, D, generator=g, device="cuda") * size
    k[:, :, 0] = 0
    k[0, :, 0] = 8
    pages, table, ks, vs = cache(K, [k], [v])
    q = (torch.randn(2, H, D, generator=g, device="cuda") * 0.01).half().float()
    q[:, :, 0] = round(logit * math.sqrt(D) * 16) / 128
    want = plain.attention([q.double().cpu()[1:]], ks, vs, [c])[0]
    for dtype in (torch.float32, torch.bfloat16):
        tol = 4 * U16 * vs[0].abs().max() + OUT_U[dtype] * want.abs() + product_step(c)
        for n_split in (0, 1, 3, 16, 20):
            out = torch.empty(1, H, D, dtype=dtype, device="cuda")
            K.kv4_decode_attention(q[1:], pages, table, dev([c]), out, n_split=n_split)
            assert ((out.double().cpu() - want).abs() <= tol).all()
            out = torch.empty(2, H, D, dtype=dtype, device="cuda")      # several rows
            K.kv4_prefill_attention(q, pages, table, dev([0, 2]), dev([c]), out, 2, n_split=n_split, tiles=False)
            assert ((out[1:].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("D,H", [(64, 1), (64, 12), (128, 4)])
@pytest.mark.parametrize("order", ["up", "down", "mixed"])
@pytest.mark.parametrize("window", [0, 150])
def test_scales_that_change_along_the_keys(K, D, H, order, window):
    """Values from 1e-4 up to f16's largest: what a warp allows its probabilities has to follow the pages."""
    c, n = 400, 3
    g = gen(H)
    size = torch.logspace(-4, math.log10(15000), c, device="cuda")
    size = {"up": size, "down": size.flip(0), "mixed": size[torch.randperm(c, generator=g, device="cuda")]}[order]
    k, v = torch.randn(c, 1, D, generator=g, device="cuda"), torch.randn(c, 1, D, generator=g, device="cuda") * size[:, None, None]
    v[c // 2, 0, :32] = torch.linspace(-65504, 65504, 32, device="cuda")      # the largest scale
    pages, table, ks, vs = cache(K, [k], [v])
    q = torch.randn(n, H, D, generator=g, device="cuda").half().float()
    sinks = torch.randn(H, generator=g, device="cuda") * 2
    for sk in (None, sinks):
        want = plain.attention([q.double().cpu()], ks, vs, [c], window=window, sinks=None if sk is None else sk.double().cpu())[0]
        for n_split in (1, 2, 5, 16):
            out = torch.empty(n, H, D, device="cuda")
            K.kv4_prefill_attention(q, pages, table, dev([0, n]), dev([c]), out, n, n_split=n_split, window=window, sinks=sk, tiles=False)
            assert ((out.double().cpu() - want).abs() <= 4 * U16 * vs[0].abs().max()).all()


@pytest.mark.parametrize("tiles", [False, True])
@pytest.mark.parametrize("size,scale", [(0.0, 0.0), (0.0, 1e-8), (0.0, 1e-30), (1e-30, 1e-12), (1e-37, 1e-6), (1e-38, 0.125)])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
def test_logits_that_vanish(K, tiles, size, scale, softcap):
    """Queries and scales so small that every logit is 0: means over the keys each row sees."""
    c, n, D = 200, 150, 64
    g = gen(2)
    pages, table, ks, vs = cache(K, [torch.randn(c, 1, D, generator=g, device="cuda")], [torch.randn(c, 1, D, generator=g, device="cuda")])
    q = torch.randn(n, 1, D, generator=g, device="cuda") * size
    out = torch.empty_like(q)
    K.kv4_prefill_attention(q, pages, table, dev([0, n]), dev([c]), out, n, tiles=tiles, scale=scale, softcap=softcap)
    hi = torch.arange(c - n + 1, c + 1)
    want = (vs[0][:, 0].cumsum(0) / torch.arange(1, c + 1)[:, None])[hi - 1]
    assert ((out[:, 0].double().cpu() - want).abs() <= 4 * U16 * vs[0].abs().max()).all()


@pytest.mark.parametrize("tiles,n_split", [(False, 1), (False, 4), (False, 20), (True, 1), (True, 3)])
def test_sinks_that_are_no_numbers_or_none(K, tiles, n_split):
    """A NaN sink makes its head NaN however the splits merge, with keys and without; one of -inf is no sink."""
    D, lens = 64, [600, 0]
    g = gen(3)
    pages, table, ks, vs = cache(K, *([torch.randn(c, 2, D, generator=g, device="cuda") for c in lens] for _ in "kv"))
    q = torch.randn(2, 4, D, generator=g, device="cuda")
    sinks = torch.tensor([math.nan, -math.inf, 0.5, math.nan], device="cuda")
    out, none = torch.empty_like(q), torch.empty_like(q)
    for o, sk in ((out, sinks), (none, None)):
        K.kv4_prefill_attention(q, pages, table, dev([0, 1, 2]), dev(lens), o, 1, tiles=tiles, n_split=n_split, sinks=sk)
    assert torch.isnan(out[:, [0, 3]]).all() and torch.equal(out[:, 1], none[:, 1])
    assert (none[1] == 0).all() and (out[1, 1:3] == 0).all()
    assert not torch.equal(out[0, 2], none[0, 2]) and torch.isfinite(out[0, 2]).all()


# ------------------------------------------------------------------------------------ arguments
@pytest.fixture(scope="module")
def small(K):
    g = gen(1)
    x = [torch.randn(40, 2, 64, generator=g, device="cuda")]
    pages, table, ks, vs = cache(K, x, x)
    return torch.randn(1, 4, 64, generator=g, device="cuda"), pages, table, dev([40]), ks, vs


@pytest.mark.parametrize("scale", [-0.125, math.nan, math.inf, 1e39])
def test_scales_that_are_none_are_refused(K, small, scale):
    q, pages, table, ctx, _, _ = small
    with pytest.raises(RuntimeError, match="scale"):
        K.kv4_decode_attention(q, pages, table, ctx, torch.empty_like(q), scale=scale)
    with pytest.raises(RuntimeError, match="scale"):
        K.kv4_prefill_attention(q, pages, table, dev([0, 1]), ctx, torch.empty_like(q), 1, scale=scale)


@pytest.mark.parametrize("tiles", [False, True])
def test_windows_beyond_32_bits(K, small, tiles):
    q, pages, table, ctx, _, _ = small
    none, some = torch.empty_like(q), torch.empty_like(q)
    K.kv4_prefill_attention(q, pages, table, dev([0, 1]), ctx, none, 1, tiles=tiles)
    for window in (-5, -2 ** 40, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 5, 2 ** 62):
        K.kv4_prefill_attention(q, pages, table, dev([0, 1]), ctx, some, 1, tiles=tiles, window=window)
        # (a window may change how the keys are shared out, and with it the last bits)
        assert ((some - none).abs() <= 1e-5).all()


@pytest.mark.parametrize("softcap", [-1.0, math.nan, math.inf, 1e39])
def test_softcaps_that_are_none_are_refused(K, small, softcap):
    q, pages, table, ctx, _, _ = small
    with pytest.raises(RuntimeError, match="softcap"):
        K.kv4_decode_attention(q, pages, table, ctx, torch.empty_like(q), softcap=softcap)
    with pytest.raises(RuntimeError, match="softcap"):
        K.token_logprobs(q[0], 64, dev([0] * 4), 0, softcap)


@pytest.mark.parametrize("n", [2 ** 31, 2 ** 32 + 1])
def test_rows_past_32_bits_are_refused(K, small, n):
    """Expanded tensors reach such counts in little memory."""
    q, pages, table, ctx, _, _ = small
    x, slot = torch.zeros(1, 2, 64, device="cuda"), dev([-1])
    with pytest.raises(RuntimeError, match="too many"):
        K.kv4_append(x.expand(n, -1, -1), x.expand(n, -1, -1), slot.expand(n), pages)
    with pytest.raises(RuntimeError, match="too many"):
        K.kv4_read(pages, slot.expand(n), 64)
    with pytest.raises(RuntimeError, match="too many"):
        K.kv4_decode_attention(q.expand(n, -1, -1), pages, table, ctx, torch.empty_like(q).expand(n, -1, -1))
    with pytest.raises(RuntimeError, match="too many"):
        K.token_logprobs(q[0, :1].expand(n, -1), 64, slot.expand(n))
    with pytest.raises(RuntimeError, match="too many"):
        K.plan_batch(dev([0]), dev([1]), table, slot.expand(n), dev([0]), 1)
