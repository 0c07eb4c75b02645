"""Token log probabilities, entropy, rank and top alternatives against 64-bit torch.

Tolerance: the sum S of up to 2e5 positive terms is added in f32 in chunks of at most 640 per lane, then
by pairs (relative error about 640 * 2^-24 at worst, random in practice), the exponentials carry 2^-22 and
the logarithm 2^-22: 1e-4 absolute bounds log S and every log probability; entropies up to 12.2 the same."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 1e-4


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def want(x, t, k):
    """x [T, V] (the values the logits hold), all on the CPU in 64 bits."""
    x = x.double().cpu()
    T, V = x.shape
    z = torch.log_softmax(x, -1)
    dead = torch.isneginf(x).all(-1)
    z[dead] = -math.inf
    p = torch.exp(z)
    ent = -(p * torch.where(p > 0, z, torch.zeros_like(z))).sum(-1)
    lp, rank = torch.zeros(T, dtype=torch.float64), torch.zeros(T, dtype=torch.int64)
    for r, c in enumerate(t.tolist()):
        if 0 <= c < V:
            lp[r] = z[r, c]
            rank[r] = 1 + (x[r] > x[r, c]).sum() + (x[r, :c] == x[r, c]).sum()
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :k]
    return lp, ent, rank, ids, z.gather(1, ids)


def check(r, w):
    lp, ent, rank, ids, top = w
    k = ids.shape[1]
    assert torch.equal(r.rank.long().cpu(), rank)
    assert torch.equal(r.top_ids.long().cpu()[:, :k], ids)
    for got, ref in ((r.logprob, lp), (r.entropy, ent), (r.top_logprobs[:, :k], top)):
        got = got.double().cpu()
        same = got == ref      # infinities
        assert (same | ((got - ref).abs() <= TOL)).all()


@pytest.mark.parametrize("T,V", [(1, 1), (1, 5), (3, 32), (2, 255), (5, 2049), (300, 1000), (1, 152064), (7, 49152), (2, 201088), (700, 4099)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("k", [0, 1, 20, 32])
def test_against_64_bits(K, T, V, dtype, k):
    g = torch.Generator(device="cuda")
    g.manual_seed(T * 7 + V)
    x = (torch.randn(T, V, generator=g, device="cuda") * 3).to(dtype)     # 16-bit types: many ties
    t = torch.randint(0, V, (T,), generator=g, device="cuda", dtype=torch.int32)
    t[0] = x[0].float().argmax()
    if T > 2:
        t[1] = -1
        t[2] = V
    r = K.token_logprobs(x, V, t, k)
    w = want(x.float(), t, min(k, V))
    check(r, w)
    if k > V:
        assert (r.top_ids[:, V:] == -1).all() and torch.isneginf(r.top_logprobs[:, V:]).all()


@pytest.mark.parametrize("order", ["up", "down", "equal", "two", "signed zeros"])
@pytest.mark.parametrize("T", [1, 600])
def test_orders_and_ties(K, order, T):
    V = 5003
    i = torch.arange(V, device="cuda", dtype=torch.float32)
    row = {"up": i * 0.01, "down": -i * 0.01, "equal": torch.full_like(i, 2.5), "two": (i % 2) * 3.0,
           "signed zeros": torch.where(i % 3 == 0, 0.0, -0.0)}[order]
    x = row[None].repeat(T, 1)
    t = (torch.arange(T, device="cuda") * 7 % V).to(torch.int32)
    r = K.token_logprobs(x, V, t, 20)
    check(r, want(x[:2], t[:2], 20) if T == 1 else want(x, t, 20))


@pytest.mark.parametrize("T", [1, 600])
def test_masked_rows(K, T):
    V = 3001
    x = torch.randn(T + 3, V, device="cuda")
    x[:, ::2] = -math.inf
    x[0] = -math.inf                    # a mask that leaves nothing
    x[1] = -math.inf
    x[1, 77] = 1.5                      # one token left
    x[2, :] = torch.finfo(torch.float32).min     # masks of the type's lowest value
    x[2, 5] = 0.0
    t = torch.randint(0, V, (T + 3,), device="cuda", dtype=torch.int32)
    t[1] = 77
    r = K.token_logprobs(x, V, t, 8)
    check(r, want(x, t, 8))
    assert r.entropy[0] == 0 and torch.isneginf(r.logprob[0]) and r.logprob[1] == 0 and r.entropy[1] == 0


def test_nan_and_infinity(K):
    x = torch.zeros(3, 3000, device="cuda")
    x[0, 2500] = math.nan
    x[1, 17] = math.inf
    r = K.token_logprobs(x, 3000, torch.zeros(3, dtype=torch.int32, device="cuda"), 2)
    assert torch.isnan(r.logprob[:2]).all() and torch.isnan(r.entropy[:2]).all()
    assert r.top_ids[1, 0] == 17 and abs(r.logprob[2].item() + math.log(3000)) < TOL


def test_strides_softcap_and_columns(K):
    g = torch.Generator(device="cuda")
    g.manual_seed(0)
    full = torch.randn(9, 4001, generator=g, device="cuda") * 40
    t = torch.arange(4, device="cuda", dtype=torch.int32) * 100
    x = full[::2][:4, 1:]       # odd row stride, no vector boundary, columns past V ignored
    r = K.token_logprobs(x, 3500, t, 5, softcap=30.0)
    y = 30.0 * torch.tanh(x[:, :3500] / 30.0)      # the kernel's 32-bit values decide ties
    lp, ent, rank, ids, top = want(30.0 * torch.tanh(x[:, :3500].double() / 30.0), t, 5)
    assert ((r.logprob.double().cpu() - lp).abs() <= TOL).all() and ((r.entropy.double().cpu() - ent).abs() <= TOL).all()
    assert ((r.top_logprobs.double().cpu() - top).abs() <= TOL).all() and y.shape == (4, 3500)


def test_repeated_calls_give_the_same_bits(K):
    x = torch.randn(3, 152064, device="cuda")
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    first = K.token_logprobs(x, 152064, t, 20)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for i in range(20):
        with torch.cuda.stream(s if i % 2 else torch.cuda.current_stream()):
            r = K.token_logprobs(x, 152064, t, 20)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_in_a_graph(K):
    x = torch.randn(2, 50000, device="cuda")
    t = torch.tensor([1, 2], dtype=torch.int32, device="cuda")
    K.token_logprobs(x, 50000, t, 3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = K.token_logprobs(x, 50000, t, 3)
    for _ in range(3):
        x.normal_()
        g.replay()
        check(r, want(x, t, 3))


def test_refusals(K):
    x, t = torch.zeros(2, 10, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="columns"):
        K.token_logprobs(x, 11, t)
    with pytest.raises(RuntimeError, match="alternatives"):
        K.token_logprobs(x, 10, t, 33)
    with pytest.raises(RuntimeError, match="targets"):
        K.token_logprobs(x, 10, t.long())
    with pytest.raises(RuntimeError, match="targets"):
        K.token_logprobs(x, 10, t[:1])
    with pytest.raises(RuntimeError, match="logits"):
        K.token_logprobs(x.t(), 2, t)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        K.token_logprobs(x.double(), 10, t)
    with pytest.raises(RuntimeError, match="logits"):
        K.token_logprobs(x.cpu(), 10, t)
