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
