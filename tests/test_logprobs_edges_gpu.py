"""Token log probabilities where they can go wrong: empty batches, infinities, what becomes of the outputs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


@pytest.mark.parametrize("k", [0, 5, 32])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_no_rows(K, k, dtype):
    r = K.token_logprobs(torch.zeros(0, 100, dtype=dtype, device="cuda"), 100, torch.zeros(0, dtype=torch.int32, device="cuda"), k)
    assert [tuple(t.shape) for t in r] == [(0,), (0,), (0,), (0, k), (0, k)]
    assert r.logprob.dtype == r.entropy.dtype == r.top_logprobs.dtype == torch.float32 and r.rank.dtype == r.top_ids.dtype == torch.int32


@pytest.mark.parametrize("V", [40, 9000, 152064])      # one warp's tile, two tiles, segments
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_rank_beside_infinities(K, V, dtype, softcap):
    """An infinite target is beaten by nothing, and equal ones go by their index like all others."""
    at = [5, 17, V - 1]
    x = torch.zeros(len(at), V, dtype=dtype, device="cuda")
    for i in at:
        x[:, i] = float("inf")
    r = K.token_logprobs(x, V, torch.tensor(at, dtype=torch.int32, device="cuda"), 4, softcap)
    assert r.rank.tolist() == [1, 2, 3] and r.top_ids[:, :3].tolist() == [at] * 3


def test_outputs_are_saved_and_kept_by_themselves(K, tmp_path):
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    x = torch.randn(3, 500, generator=g, device="cuda")
    r = K.token_logprobs(x, 500, torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), 4)
    torch.save(tuple(r), tmp_path / "r.pt")
    assert all(torch.equal(a, b) for a, b in zip(r, torch.load(tmp_path / "r.pt")))
    assert all(t.untyped_storage().nbytes() == t.numel() * 4 for t in r)


@pytest.mark.parametrize("V", [300, 5000, 60000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_ranks_and_alternatives_under_a_softcap(K, V, dtype):
    """Logits that the cap leaves apart: their order is that of the logits.  Equal logits stay equal."""
    g = torch.Generator(device="cuda")
    g.manual_seed(V)
    T, k = 6, 20
    # multiples of 1/4 around 110 (bf16 rounds some alike), where the cap has a slope of 0.02 and more; the rest far below
    x = torch.full((T, V), -40.0, device="cuda")
    for r in range(T):
        at = torch.randperm(V, generator=g, device="cuda")[:100]
        x[r, at] = torch.randperm(100, generator=g, device="cuda").float() / 4 + 100
    x = x.to(dtype)
    order = torch.sort(x.double().cpu(), dim=-1, descending=True, stable=True).indices
    t = torch.stack([order[r, 7 * r] for r in range(T)]).to(torch.int32).cuda()
    r = K.token_logprobs(x, V, t, k, softcap=50.0)
    assert torch.equal(r.top_ids.long().cpu(), order[:, :k])
    same = torch.stack([(x[i] == x[i, t[i].long()]).cpu()[:t[i]].sum() for i in range(T)])
    assert r.rank.tolist() == [1 + int((x[i] > x[i, t[i].long()]).sum()) + int(same[i]) for i in range(T)]
