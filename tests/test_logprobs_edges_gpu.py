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
