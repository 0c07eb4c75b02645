"""4-bit KV cache on the GPU: append and read against the formulas in 64 bits, attention against a plain
softmax over the values the bytes stand for.

Tolerance of attention, from the kernel's roundings (u = 2^-11, f16): a probability is rounded to f16, its
product with a scale once more, and the denominator sums rounded probabilities: 3 u of the largest |v|,
plus 1 u for the f32 sums, the exponentials and probabilities below f16's range, plus the output's own
rounding.  Chunks of many rows round probabilities and values to bf16 instead (2^-8): 4 * 2^-8."""
import math

import numpy as np
import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu
U16, UBF = 2.0 ** -11, 2.0 ** -8
OUT_U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def random_rows(g, shape, dtype=torch.bfloat16):
    x = torch.randn(shape, generator=g, device="cuda") + 0.5 * torch.randn(shape[-1], generator=g, device="cuda")
    return x.to(dtype)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,Hkv,form", [(1, 1, "rows"), (17, 3, "slices"), (50, 2, "odd"), (33, 4, "pages")])
def test_append_reads_back_the_formula(K, D, dtype, T, Hkv, form):
    g = gen(T + D)
    base = random_rows(g, (2, 64, 2 * Hkv + 1, D))    # bf16 values: their codes are the same in 32 and 64 bits
    if form == "rows":
        k, v = (base[i, :T, :Hkv].contiguous().to(dtype) for i in (0, 1))
    elif form == "slices":
        both = base[0].to(dtype)
        k, v = both[:T, 1:1 + Hkv], both[:T, 1 + Hkv:]
    elif form == "odd":       # rows that start on no vector boundary
        flat = torch.zeros(2, 64, 2 * Hkv, D + 1, dtype=dtype, device="cuda")
        flat[..., 1:] = base[:, :, :2 * Hkv].to(dtype)
        k, v = flat[0, :T, :Hkv, 1:], flat[1, :T, Hkv:, 1:]
    else:                     # the pages of a 16-bit cache
        pg = base[:, :, :Hkv].reshape(2, 4, 16, Hkv, D).transpose(2, 3).contiguous().to(dtype)
        k, v = pg[0], pg[1]
    P = 9
    slot = torch.randperm(P * 16, generator=g, device="cuda")[:T].to(torch.int32)
    if T > 4:
        slot[3] = -1
    before = torch.randint(0, 256, (P, Hkv, K.kv4_page_bytes(D)), generator=g, device="cuda", dtype=torch.uint8)
    pages = before.clone()
    K.kv4_append(k, v, slot, pages)
    rk, rv = K.kv4_read(pages, slot, D, torch.float32)
    if form == "pages":
        k, v = (x.transpose(1, 2).reshape(64, Hkv, D)[:T] for x in (k, v))
    live = (slot >= 0).cpu().numpy()
    got_k, got_v = plain.values(pages.cpu().numpy(), D)       # [P, Hkv, 16, D]
    old_k, old_v = plain.values(before.cpu().numpy(), D)
    sl = slot.cpu().numpy()
    written = np.zeros(P * 16, bool)
    written[sl[live]] = True
    for x, r, got, old in ((k, rk, got_k, old_k), (v, rv, got_v, old_v)):
        want, _ = plain.quantized(x.double().cpu().numpy())
        want[~live] = 0
        np.testing.assert_array_equal(r.double().cpu().numpy(), want.astype(np.float32).astype(np.float64))
        rows = got.transpose(0, 2, 1, 3).reshape(P * 16, Hkv, D)
        np.testing.assert_array_equal(rows[sl[live]], want[live])
        np.testing.assert_array_equal(rows[~written], old.transpose(0, 2, 1, 3).reshape(P * 16, Hkv, D)[~written])


def test_append_error_bound_of_float32(K):
    g = gen(5)
    k = torch.randn(200, 2, 128, generator=g, device="cuda") * torch.logspace(-4, 3, 200, device="cuda")[:, None, None]
    pages = torch.zeros(13, 2, K.kv4_page_bytes(128), dtype=torch.uint8, device="cuda")
    slot = torch.arange(200, dtype=torch.int32, device="cuda")
    K.kv4_append(k, -k, slot, pages)
    rk, rv = K.kv4_read(pages, slot, 128, torch.float32)
    grp = k.reshape(200, 2, 4, 32)
    lo, step = grp.amin(-1, keepdim=True).abs(), (grp.amax(-1, keepdim=True) - grp.amin(-1, keepdim=True)) / 15
    # half a step, the rounding of the scale over 15 steps and of the minimum (u each, and f16's smallest step)
    bound = 0.5 * step * (1 + 2 * U16) + 15 * step * U16 + 2 * (lo + 15 * step) * U16 + 16 * 2.0 ** -24
    assert ((rk.reshape(200, 2, 4, 32) - grp).abs() <= bound).all()
    hi = (-grp).amin(-1, keepdim=True).abs()
    bound = 0.5 * step * (1 + 2 * U16) + 15 * step * U16 + 2 * (hi + 15 * step) * U16 + 16 * 2.0 ** -24
    assert ((rv.reshape(200, 2, 4, 32) + grp).abs() <= bound).all()


def test_append_constants_infinities_nan(K):
    k = torch.zeros(5, 1, 64, device="cuda")
    k[0] = 3.0
    k[1, 0, 3] = math.inf
    k[2, 0, 40] = -math.inf
    k[3, 0, 1] = math.nan
    k[4, 0, :32] = 1e30
    pages = torch.full((1, 1, K.kv4_page_bytes(64)), 255, dtype=torch.uint8, device="cuda")
    slot = torch.arange(5, dtype=torch.int32, device="cuda")
    K.kv4_append(k, k, slot, pages)
    for r in K.kv4_read(pages, slot, 64, torch.float32):
        r = r[:, 0].cpu()
        assert (r[0] == 3).all()
        assert r[1, 3] > 65000 and torch.isfinite(r[1]).all() and (r[1, 32:] == 0).all()
        assert r[2, 40] == -65504 and (r[2, :32] == 0).all()
        assert torch.isnan(r[3, :32]).all() and (r[3, 32:] == 0).all()
        assert (r[4, :32] == 65504).all() and (r[4, 32:] == 0).all()


def test_append_slot_past_the_pages_is_reported(K):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.register_error_word(err.device, err)
    try:
        pages = torch.zeros(2, 1, K.kv4_page_bytes(64), dtype=torch.uint8, device="cuda")
        x = torch.ones(1, 1, 64, device="cuda")
        K.kv4_append(x, x, torch.tensor([32], dtype=torch.int32, device="cuda"), pages)
        assert err.item() == 2 and (pages == 0).all()
    finally:
        K.register_error_word(err.device, None)


# ------------------------------------------------------------------------------------ attention
def cache_of(K, g, lens, Hkv, D, wide=None):
    """A cache holding random rows of the given lengths: pages, table, and the values (64 bits)."""
    n = [max(1, -(-c // 16)) for c in lens]
    P, width = sum(n) + 3, max(n) + 1
    pages = torch.full((P, Hkv, K.kv4_page_bytes(D)), 255, dtype=torch.uint8, device="cuda")   # NaN scales everywhere
    ids = (torch.randperm(P - 1, generator=g, device="cuda") + 1).to(torch.int32)
    table = torch.zeros(len(lens), width, dtype=torch.int32, device="cuda")
    at, ks, vs = 0, [], []
    for b, c in enumerate(lens):
        table[b, :n[b]] = ids[at:at + n[b]]
        at += n[b]
        k, v = random_rows(g, (c, Hkv, D)), random_rows(g, (c, Hkv, D))
        if wide is not None and c:
            k[:, :, 3] *= wide
        j = torch.arange(c, device="cuda")
        slot = (table[b, j // 16] * 16 + j % 16).to(torch.int32)
        K.kv4_append(k, v, slot, pages)
        rk, rv = K.kv4_read(pages, slot, D, torch.float32)
        ks.append(rk.double().cpu())
        vs.append(rv.double().cpu())
    return pages, table, ks, vs


DEC = [  # lens, H, Hkv, D
    ([1], 1, 1, 64), ([16, 17, 15, 1, 0, 100], 8, 2, 64), ([33], 28, 4, 128), ([1000, 7, 250], 7, 1, 128),
    ([300, 41], 16, 1, 128), ([77], 40, 2, 128), ([129, 500], 71, 1, 64), ([64, 65], 9, 3, 64),
]


@pytest.mark.parametrize("lens,H,Hkv,D", DEC)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n_split", [0, 1, 3])
def test_decode(K, lens, H, Hkv, D, dtype, n_split):
    g = gen(len(lens) * 100 + H)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    q = (torch.randn(len(lens), H, D, generator=g, device="cuda") * 1.5).to(torch.float16 if dtype == torch.float32 else dtype).to(dtype)
    out = torch.full_like(q, math.nan)
    K.kv4_decode_attention(q, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, n_split=n_split)
    want = plain.attention([r[None] for r in q.double().cpu()], ks, vs, lens)
    for b, c in enumerate(lens):
        w = want[b][0]
        if c == 0:
            assert (out[b] == 0).all()
        else:
            tol = 4 * U16 * vs[b].abs().max() + OUT_U[dtype] * w.abs()
            assert ((out[b].double().cpu() - w).abs() <= tol).all()


@pytest.mark.parametrize("window", [1, 16, 40, 5000])
@pytest.mark.parametrize("softcap", [0.0, 20.0])
@pytest.mark.parametrize("sink", [False, True])
def test_decode_window_softcap_sinks(K, window, softcap, sink):
    lens, H, Hkv, D = [5, 200, 48, 1], 8, 2, 64
    g = gen(window)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    q = torch.randn(4, H, D, generator=g, device="cuda") .to(torch.bfloat16)
    sinks = torch.randn(H, generator=g, device="cuda") * 3 if sink else None
    want = plain.attention([r[None] for r in q.double().cpu()], ks, vs, lens, window=window, softcap=softcap, scale=0.3,
                           sinks=sinks.double().cpu() if sink else None)
    for n_split in (1, 4):
        out = torch.empty(4, H, D, device="cuda")
        K.kv4_decode_attention(q, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, window=window,
                               softcap=softcap, scale=0.3, sinks=sinks, n_split=n_split)
        for b in range(4):
            assert ((out[b].double().cpu() - want[b][0]).abs() <= 4 * U16 * vs[b].abs().max()).all()


def test_decode_wide_keys_and_tiny_queries(K):
    """Logits of hundreds (one key takes all), and queries far below f16's range."""
    lens, H, Hkv, D = [90, 33], 4, 2, 128
    g = gen(3)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D, wide=200)
    for size, scale in ((8.0, 0.0), (1e-20, 1e20)):
        q = torch.randn(2, H, D, generator=g, device="cuda").to(torch.bfloat16).float() * size
        q = q.to(torch.bfloat16)
        out = torch.empty(2, H, D, device="cuda")
        K.kv4_decode_attention(q, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, scale=scale)
        want = plain.attention([r[None] for r in q.double().cpu()], ks, vs, lens, scale=scale or None)
        zmax = max((ks[b].abs().max() * q[b].double().abs().max().item() * D * (scale or D ** -0.5)) for b in range(2))
        for b in range(2):
            # logits up to zmax carry an f32 rounding each (2^-22 of their size, in all)
            tol = (4 * U16 + 2 * 2.0 ** -22 * zmax) * vs[b].abs().max()
            assert ((out[b].double().cpu() - want[b][0]).abs() <= tol).all()


def test_decode_uniform_long_context(K):
    """Equal logits over many keys: the mean of the values."""
    c, D = 5001, 64
    g = gen(9)
    pages, table, ks, vs = cache_of(K, g, [c], 1, D)
    out = torch.empty(1, 2, D, device="cuda")
    q = torch.zeros(1, 2, D, device="cuda")
    K.kv4_decode_attention(q, pages, table, torch.tensor([c], dtype=torch.int32, device="cuda"), out)
    assert ((out[0, 0].double().cpu() - vs[0].mean(0)[0]).abs() <= 4 * U16 * vs[0].abs().mean()).all()


def test_decode_nan_value_beyond_the_window_is_not_read(K):
    lens, D = [40], 64
    g = gen(1)
    pages, table, ks, vs = cache_of(K, g, lens, 1, D)
    bad = torch.full((1, 1, D), math.nan, device="cuda")
    K.kv4_append(bad, bad, (table[0, 1:2] * 16 + 4).to(torch.int32), pages)   # key 20
    q = torch.randn(1, 2, D, generator=g, device="cuda")
    out = torch.empty(1, 2, D, device="cuda")
    K.kv4_decode_attention(q, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, window=19)
    assert torch.isfinite(out).all()      # keys 21 .. 39
    K.kv4_decode_attention(q, pages, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), out, window=20)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("lens,n_split", [([1], 1), ([17], 4), ([200], 16), ([200], 20)])
def test_decode_all_keys_nan(K, lens, n_split):
    """No finite logit anywhere is not the same as no key."""
    g = gen(1)
    pages, table, ks, vs = cache_of(K, g, lens, 1, 64)
    j = torch.arange(lens[0], device="cuda")
    bad = torch.full((lens[0], 1, 64), math.nan, device="cuda")
    K.kv4_append(bad, bad, (table[0, j // 16] * 16 + j % 16).to(torch.int32), pages)
    out = torch.zeros(1, 2, 64, device="cuda")
    K.kv4_decode_attention(torch.randn(1, 2, 64, device="cuda"), pages, table,
                           torch.tensor(lens, dtype=torch.int32, device="cuda"), out, n_split=n_split)
    assert torch.isnan(out).all()


@pytest.mark.parametrize("H,Hkv,D", [(28, 4, 128), (16, 2, 64), (24, 1, 128)])
@pytest.mark.parametrize("sink", [False, True])
def test_decode_splits_merge_alike_in_clusters_and_in_memory(K, H, Hkv, D, sink):
    """2 to 16 splits merge in a cluster while their CTAs are all resident, else through memory: a sequence's
    bits are the same, alone (clusters) and in a batch of 40 (memory)."""
    g = gen(8)
    lens = [700, 33, 1, 250] * 10
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(40, H, D, generator=g, device="cuda").to(torch.bfloat16)
    sinks = torch.randn(H, generator=g, device="cuda") if sink else None
    for n_split in (2, 8, 16):
        every, one = torch.empty(40, H, D, device="cuda"), torch.empty(1, H, D, device="cuda")
        K.kv4_decode_attention(q, pages, table, ctx, every, n_split=n_split, sinks=sinks)
        for b in range(5):
            K.kv4_decode_attention(q[b:b + 1], pages, table[b:b + 1], ctx[b:b + 1], one, n_split=n_split, sinks=sinks)
            assert torch.equal(one[0], every[b])


def test_decode_strides_and_streams(K):
    lens, H, Hkv, D = [50, 20], 8, 2, 64
    g = gen(2)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    big = torch.randn(2, 3 * H, D, generator=g, device="cuda").to(torch.bfloat16)
    q = big[:, H:2 * H]
    ref = torch.empty(2, H, D, dtype=torch.bfloat16, device="cuda")
    K.kv4_decode_attention(q.contiguous(), pages, table, ctx, ref)
    buf = torch.zeros(2, H, 2 * D, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        K.kv4_decode_attention(q, pages, table, ctx, buf[:, :, D:])
    s.synchronize()
    assert torch.equal(buf[:, :, D:], ref) and (buf[:, :, :D] == 0).all()


def test_decode_fixed_splits_do_not_depend_on_the_batch(K):
    lens, H, Hkv, D = [700, 300, 1, 90], 8, 2, 128
    g = gen(4)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    q = torch.randn(4, H, D, generator=g, device="cuda").to(torch.bfloat16)
    all4, one = torch.empty(4, H, D, device="cuda"), torch.empty(1, H, D, device="cuda")
    K.kv4_decode_attention(q, pages, table, ctx, all4, n_split=8)
    for b in range(4):
        K.kv4_decode_attention(q[b:b + 1], pages, table[b:b + 1], ctx[b:b + 1], one, n_split=8)
        assert torch.equal(one[0], all4[b])


PRE = [  # cached, new, H, Hkv, D
    ([0], [1], 1, 1, 64), ([0, 5, 30], [3, 0, 17], 8, 2, 64), ([100], [33], 28, 4, 128), ([0, 16, 250], [40, 1, 70], 7, 1, 128),
    ([3, 0], [150, 0], 16, 2, 128), ([60], [200], 9, 3, 64), ([11, 400, 0], [129, 64, 300], 8, 8, 128),
]


@pytest.mark.parametrize("old,new,H,Hkv,D", PRE)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("window", [0, 37])
def test_prefill(K, old, new, H, Hkv, D, dtype, window):
    lens = [a + n for a, n in zip(old, new)]
    g = gen(sum(new) + H)
    pages, table, ks, vs = cache_of(K, g, lens, Hkv, D)
    T = sum(new)
    q = torch.randn(T + 2, H, D, generator=g, device="cuda").to(dtype)
    off = np.concatenate([[0], np.cumsum(new)])
    out = torch.full_like(q, 7)
    K.kv4_prefill_attention(q, pages, table, torch.tensor(off, dtype=torch.int32, device="cuda"),
                            torch.tensor(lens, dtype=torch.int32, device="cuda"), out, max(new), window=window)
    want = plain.attention([q[off[b]:off[b + 1]].double().cpu() for b in range(len(new))], ks, vs, lens, window=window)
    for b in range(len(new)):
        if new[b]:
            tol = 4 * UBF * vs[b].abs().max() + OUT_U[dtype] * want[b].abs()
            assert ((out[off[b]:off[b + 1]].double().cpu() - want[b]).abs() <= tol).all()
    assert (out[T:] == 7).all()


def test_prefill_splits_the_blocks_of_a_short_last_wave(K):
    """Two blocks more than multiprocessors: the last two sequences' keys are split, the others' are not."""
    g = gen(77)
    B = torch.cuda.get_device_properties(0).multi_processor_count + 2
    lens = [66 + b % 40 for b in range(B - 2)] + [2190, 1500]
    pages, table, ks, vs = cache_of(K, g, lens, 1, 64)
    new = [66] * B
    q = torch.randn(sum(new), 1, 64, generator=g, device="cuda").to(torch.bfloat16)
    off = torch.arange(0, sum(new) + 1, 66, dtype=torch.int32, device="cuda")
    ctx = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out, one = torch.full_like(q, 7), torch.full_like(q, 7)
    K.kv4_prefill_attention(q, pages, table, off, ctx, out, 66)
    K.kv4_prefill_attention(q, pages, table, off, ctx, one, 66, n_split=1)
    assert torch.equal(out[:66 * (B - 2)], one[:66 * (B - 2)])
    for b in (0, 1, B - 3, B - 2, B - 1):
        want = plain.attention([q[66 * b:66 * b + 66].double().cpu()], ks[b:b + 1], vs[b:b + 1], lens[b:b + 1])[0]
        tol = 4 * UBF * vs[b].abs().max() + OUT_U[torch.bfloat16] * want.abs()
        for o in (out, one):
            assert ((o[66 * b:66 * b + 66].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("tiles", [False, True])
def test_context_past_the_table_is_reported(K, tiles):
    g = gen(5)
    pages, table, ks, vs = cache_of(K, g, [30], 1, 64)          # three table columns, the last a page of zeros' id
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.register_error_word(err.device, err)
    try:
        q = torch.randn(1, 1, 64, generator=g, device="cuda").to(torch.bfloat16)
        off = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
        K.kv4_prefill_attention(q, pages, table, off, torch.tensor([48], dtype=torch.int32, device="cuda"), torch.empty_like(q), 1, tiles=tiles)
        assert err.item() == 0
        K.kv4_prefill_attention(q, pages, table, off, torch.tensor([49], dtype=torch.int32, device="cuda"), torch.empty_like(q), 1, tiles=tiles)
        assert err.item() == 2
    finally:
        K.register_error_word(err.device, None)


def test_refusals(K):
    pages = torch.zeros(4, 2, K.kv4_page_bytes(64), dtype=torch.uint8, device="cuda")
    q = torch.zeros(1, 4, 64, device="cuda")
    table, ctx = torch.zeros(1, 2, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    out = torch.empty_like(q)
    with pytest.raises(RuntimeError, match="query heads"):
        K.kv4_decode_attention(q[:, :3], pages, table, ctx, out[:, :3])
    with pytest.raises(RuntimeError, match="q is"):
        K.kv4_decode_attention(torch.zeros(1, 4, 128, device="cuda"), pages, table, ctx, torch.zeros(1, 4, 128, device="cuda"))
    with pytest.raises(RuntimeError, match="queries for"):
        K.kv4_decode_attention(torch.zeros(2, 4, 64, device="cuda"), pages, table, ctx, torch.zeros(2, 4, 64, device="cuda"))
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        K.kv4_decode_attention(q.double(), pages, table, ctx, out)
    with pytest.raises(RuntimeError, match="bytes per page"):
        K.kv4_decode_attention(q, torch.zeros(4, 2, 100, dtype=torch.uint8, device="cuda"), table, ctx, out)
    with pytest.raises(RuntimeError, match="int32"):
        K.kv4_decode_attention(q, pages, table.long(), ctx, out)
    with pytest.raises(RuntimeError, match="workspace"):
        K.kv4_decode_attention(q, pages, torch.zeros(1, 64, dtype=torch.int32, device="cuda"), ctx, out, n_split=20,
                               workspace=torch.zeros(8, device="cuda"))
    with pytest.raises(RuntimeError, match="max_new"):
        K.kv4_prefill_attention(q, pages, table, torch.zeros(2, dtype=torch.int32, device="cuda"), ctx, out, 2)
    x = torch.zeros(3, 2, 64, device="cuda")
    slot = torch.zeros(3, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="heads of"):
        K.kv4_append(x[:, :1], x[:, :1], slot, pages)
    with pytest.raises(RuntimeError, match="rows for"):
        K.kv4_append(x[:2], x[:2], slot, pages)
    with pytest.raises(RuntimeError, match="differ in type"):
        K.kv4_append(x, x.half(), slot, pages)
    with pytest.raises(RuntimeError, match="heads of"):
        K.kv4_read(pages, slot, 128)
    with pytest.raises(ValueError):
        K.kv4_page_bytes(96)
