"""Scoring and the engine on a 4-bit KV cache where they can go wrong."""
import numpy as np
import pytest
import torch

from fak_b200.config import EngineConfig, preset
from fak_b200.gguf.synth import write_synthetic_gguf

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module", params=["tiny-qwen2", "tiny-llama", "tiny-gemma2"])
def model_file(request, tmp_path_factory):
    path = str(tmp_path_factory.mktemp("kv4e") / f"{request.param}.gguf")
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


@pytest.mark.parametrize("precision", ["bf16", "q4"])
def test_score_refuses_tokens_outside_the_vocabulary(model_file, precision):
    """Before they reach the device, whose error word would end every request that runs."""
    eng = engine(model_file, precision)
    V = eng.cfg.vocab_size
    p = prompts(V, [30])[0]
    alone = eng.generate([p], max_new_tokens=8)[0]
    r = eng.add_request(p, 8)
    eng.step()
    for bad in ([[1, V]], [[1, 2], [3, -1, 4]]):
        with pytest.raises(ValueError, match="vocabulary"):
            eng.score(bad)
    while eng.has_work():
        eng.step()
    assert r.finish_reason == "length" and r.output == alone
    assert len(eng.score([[0, V - 1]])[0]["logprob"]) == 1


@pytest.mark.parametrize("held", [False, True])
def test_score_groups_prompts_beside_a_full_prefix_cache(model_file, held):
    """Cached prefixes that nobody uses give way to a chunk's prompts, so that a pool full of them does not mean
    one prompt a pass; prefixes that a running request holds stay."""
    ps = prompts(preset("tiny-llama").vocab_size, [40] * 8, 1)
    want = engine(model_file).score(ps)
    eng = engine(model_file, kv_pages=64, max_prefill_tokens=512)
    seen = prompts(eng.cfg.vocab_size, [200] * 4, 2)
    for p in seen:
        eng.generate([p], max_new_tokens=4)
    assert eng.pool.n_free() < 24       # the prompts take 24 pages
    if held:
        reqs = [eng.add_request(p + [1], 40) for p in seen]
        while any(not r.output for r in reqs):
            eng.step()
    calls, plain = [], eng.runner.score

    def score(*a, **kw):
        calls.append(1)
        return plain(*a, **kw)
    eng.runner.score = score
    got = eng.score(ps)
    assert (len(calls) > 1) if held else (len(calls) == 1)
    for a, b in zip(want, got):     # the same values through other tiles, as in chunks
        np.testing.assert_allclose(a["logprob"], b["logprob"], atol=0.1)
    if held:
        while eng.has_work():
            eng.step()
        assert all(r.finish_reason == "length" for r in reqs)


@pytest.mark.parametrize("graphs", [False, True])
def test_poisoned_scratch_and_pages_change_nothing(model_file, graphs):
    """The debug fill: NaN in the scratch of the 4-bit path too, 32768 wherever a page was not written."""
    from fak_b200.ops import kernels as K
    eng = engine(model_file, graphs=graphs, debug_poison=True)
    ps = prompts(eng.cfg.vocab_size, [40, 7, 100, 16], 2)
    rn = eng.runner
    k, v = K.kv4_read(rn.kv.pages[0], torch.arange(64, dtype=torch.int32, device="cuda") + 160, rn.D, torch.float32)
    assert (k == 32768).all() and (v == 32768).all()
    if not graphs:      # (their capture runs steps)
        assert all(torch.isnan(t).all() for t in (rn.stage.k, rn.stage.v, rn.attn_out, rn.kv4_ws))
    clean = engine(model_file, graphs=graphs)
    assert eng.generate(ps, max_new_tokens=24) == clean.generate(ps, max_new_tokens=24)
    assert eng.score(ps, top_k=2) == clean.score(ps, top_k=2)


@pytest.mark.parametrize("precision", ["bf16", "q4"])
def test_score_in_chunks_of_either_cache(model_file, precision):
    """Chunks in which some prompts have no token left, or none yet."""
    ps = prompts(preset("tiny-llama").vocab_size, [100, 3, 61, 20, 1], 1)
    whole = engine(model_file, precision).score(ps, top_k=3)
    for cap in (17, 32):
        for a, b in zip(whole, engine(model_file, precision, max_prefill_tokens=cap).score(ps, top_k=3)):
            # the same values through other tiles: 16-bit roundings of the attention and GEMM inputs move
            assert len(a["logprob"]) == len(b["logprob"])
            np.testing.assert_allclose(a["logprob"], b["logprob"], atol=0.1)
            np.testing.assert_allclose(a["entropy"], b["entropy"], atol=0.1)


@pytest.mark.parametrize("drafter", ["self", "lookup", "multi"])
def test_speculation_keeps_the_tokens(model_file, drafter):
    """Verified tokens are those of one step after another, drafts and their rejected rows in the pages or not."""
    p = prompts(preset("tiny-llama").vocab_size, [11, 40], 6)
    ps = [p[0] * 4, p[1]]       # one that repeats itself
    want = engine(model_file, graphs=True).generate(ps, max_new_tokens=24)
    eng = engine(model_file, graphs=True, spec_k=3, spec_drafter=drafter, max_batch=16)    # 4 rows a request
    assert eng.generate(ps, max_new_tokens=24) == want
    assert eng.stats["spec_proposed"] > 0


@pytest.mark.parametrize("precision", [None, "q4"])
def test_the_benchmark_names_the_cache_it_ran_on(precision):
    import json
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    env = {k: v for k, v in os.environ.items() if k != "FAK_KV_PRECISION"}
    if precision:
        env["FAK_KV_PRECISION"] = precision
    r = subprocess.run([sys.executable, "bench.py", "--model", "tiny-qwen2", "--mix", "q8_0", "--steps", "1", "--warmup", "3", "--agents", "2",
                        "--prefix", "64", "--user", "16", "--decode", "4"], cwd=root, env=env, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
    line = json.loads(r.stdout.strip().splitlines()[-1])
    assert line["config"]["kv_dtype"] == (precision or "bf16") and line["value"] > 0
