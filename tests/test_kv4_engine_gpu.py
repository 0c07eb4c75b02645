"""The engine on a 4-bit KV cache, and scoring (plan, append, attention and log probabilities together)."""
import numpy as np
import pytest
import torch

from fak_b200.config import EngineConfig, preset
from fak_b200.gguf.synth import write_synthetic_gguf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["tiny-qwen2", "tiny-llama", "tiny-gemma2"])
def model_file(request, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("kv4") / f"{request.param}.gguf")
    write_synthetic_gguf(path, preset(request.param), "q8_0", seed=5, std=0.05)
    return path


def engine(path, precision="q4", graphs=False, **kw):
    from fak_b200.engine import Engine
    kw = {"max_batch": 4, "kv_pages": 256, **kw}
    eng = Engine.from_gguf(path, EngineConfig(cuda_graph=graphs, graph_batch_buckets=(1, 2, 4), kv_precision=precision, **kw),
                           "cuda", max_context=1024)
    if graphs:
        eng.warmup_graphs()
    return eng


def prompts(vocab, lens, seed=0):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, vocab, n).tolist() for n in lens]


def logprobs(logits, p):
    z = torch.log_softmax(logits.double(), -1)
    return z, z[:-1].gather(1, torch.tensor(p[1:], device=z.device)[:, None])[:, 0]


@pytest.mark.parametrize("precision,bound", [("bf16", 0.2), ("q4", 0.4)])
def test_score_against_the_reference(model_file, precision, bound):
    """Other engine tests hold logits to a cosine of 0.995 with the fp32 reference: an error of 0.1 of their
    size, so 0.2 of it in a log probability on average.  4-bit keys and values (groups of 32 normal values
    span about 4 sigma: a step of 0.27 sigma, rms error 0.08) may double that."""
    from fak_b200.models.reference import ReferenceModel
    ref = ReferenceModel.from_gguf(model_file, "cuda")
    eng = engine(model_file, precision)
    ps = prompts(eng.cfg.vocab_size, [33, 2, 90])
    for p, r in zip(ps, eng.score(ps, top_k=3)):
        logits = ref.forward(torch.tensor(p))
        z, want = logprobs(logits, p)
        size = (logits - logits.mean(-1, keepdim=True)).pow(2).mean().sqrt().item()
        got = torch.tensor(r["logprob"], device="cuda", dtype=torch.float64)
        assert got.shape == want.shape and (got - want).abs().mean().item() <= bound * size
        assert len(r["entropy"]) == len(p) and len(r["rank"]) == len(p) - 1 and len(r["top_ids"]) == len(p)


@pytest.mark.parametrize("precision", ["bf16", "q4"])
def test_score_is_the_logits_score(model_file, precision):
    """Against log_softmax of the same logits in 64 bits, rows of every prompt in their places."""
    eng = engine(model_file, precision)
    ps = prompts(eng.cfg.vocab_size, [5, 40, 17], 3)
    kept = []
    from fak_b200.ops import kernels as K
    plain = K.token_logprobs

    def keep(logits, V, targets, k=0, softcap=0.0):
        x = logits[:, :V].double()
        kept.append(softcap * torch.tanh(x / softcap) if softcap else x)
        return plain(logits, V, targets, k, softcap)
    K.token_logprobs = keep
    try:
        res = eng.score(ps, top_k=4)
    finally:
        K.token_logprobs = plain
    rows = torch.cat(kept)
    at = 0
    for p, r in zip(ps, res):
        z, want = logprobs(rows[at:at + len(p)], p)
        at += len(p)
        np.testing.assert_allclose(r["logprob"], want.cpu().numpy(), atol=1e-4)
        np.testing.assert_allclose(r["entropy"], -(z.exp() * z).sum(-1).cpu().numpy(), atol=1e-4)
        top = z.topk(4, -1)
        np.testing.assert_allclose(r["top_logprobs"], top.values.cpu().numpy(), atol=1e-4)
        for i, t in enumerate(p[1:]):
            assert r["rank"][i] == 1 + int((rows[at - len(p) + i] > rows[at - len(p) + i, t]).sum()) or \
                (rows[at - len(p) + i] == rows[at - len(p) + i, t]).sum() > 1
    assert eng.pool.n_free() == 255


def test_score_in_chunks(model_file):
    """A chunk limit below the prompts' lengths: later chunks attend to earlier ones through the pages."""
    ps = prompts(preset("tiny-llama").vocab_size, [100, 3, 61, 20], 1)
    whole = engine(model_file).score(ps)
    parts = engine(model_file, max_prefill_tokens=32).score(ps)
    few_pages = engine(model_file, kv_pages=9).score(ps)       # groups of prompts whose pages fit
    for a, b, c in zip(whole, parts, few_pages):
        # the same values through other tiles: f16 / bf16 roundings of the attention and GEMM inputs move
        np.testing.assert_allclose(a["logprob"], b["logprob"], atol=0.1)
        np.testing.assert_allclose(a["logprob"], c["logprob"], atol=0.1)


def test_generate_batch_and_graphs_agree(model_file):
    eng, gr = engine(model_file), engine(model_file, graphs=True)
    ps = prompts(eng.cfg.vocab_size, [40, 7, 100, 16], 2)
    alone = [eng.generate([p], max_new_tokens=24)[0] for p in ps]
    assert gr.generate(ps, max_new_tokens=24) == alone
    assert all(len(o) == 24 for o in alone)


def test_generate_reuses_prefixes(model_file):
    eng = engine(model_file, graphs=True)
    p = prompts(eng.cfg.vocab_size, [80], 4)[0]
    a = eng.generate([p + [1, 2, 3]], max_new_tokens=8)[0]
    before = eng.stats["prefill_tokens_avoided"]
    assert eng.generate([p + [1, 2, 3]], max_new_tokens=8)[0] == a
    assert eng.stats["prefill_tokens_avoided"] > before


def test_refusals(model_file):
    from fak_b200.engine.disagg import prefill_handoffs
    with pytest.raises(ValueError, match="bf16 or q4"):
        engine(model_file, "int3")
    with pytest.raises(NotImplementedError, match="swap"):
        engine(model_file, preempt_mode="swap")
    with pytest.raises(NotImplementedError, match="tree"):
        engine(model_file, spec_k=2, spec_drafter="tree")
    eng = engine(model_file)
    with pytest.raises(NotImplementedError, match="hand-off"):
        prefill_handoffs(eng, [[1, 2]])
    with pytest.raises(NotImplementedError, match="span eviction"):
        eng.evict_span(None, 0, 1)
    with pytest.raises(ValueError, match="empty"):
        eng.score([[1], []])
    with pytest.raises(ValueError, match="context"):
        eng.score([[1] * 2000])
    with pytest.raises(ValueError, match="alternatives"):
        eng.score([[1, 2]], top_k=33)
