"""What of the 4-bit cache and scoring needs no GPU: configuration, planning, argument checks, the layout."""
import numpy as np
import pytest
import torch

import kv4_plain as plain
from fak_b200.config import EngineConfig, preset


def test_capacity_tier():
    from fak_b200.capacity import kv_bytes_per_token, parse_kv_precision
    from fak_b200.models.runner import KV4Cache, KVCache
    cfg = preset("qwen2.5-7b")
    assert parse_kv_precision("q4") == "q4"
    per = KV4Cache.bytes_per_page(cfg.n_layers, cfg.n_kv_heads, cfg.head_dim)
    assert per == 16 * kv_bytes_per_token(cfg, precision="q4")
    assert KVCache.bytes_per_page(cfg.n_layers, cfg.n_kv_heads, cfg.head_dim) == per * 32 // 10


def test_env_and_cli(monkeypatch):
    from fak_b200 import cli
    monkeypatch.setenv("FAK_KV_PRECISION", "q4")
    assert EngineConfig.from_env().kv_precision == "q4"
    with pytest.raises(SystemExit):
        cli.main(["score", "--kv-precision", "int4", "text"])
    with pytest.raises(SystemExit, match="GPU engine"):
        cli.main(["score", "--cpu", "text"])


def test_cache_shapes_and_refusals():
    from fak_b200.models.runner import KV4Cache
    from fak_b200.ops import kernels as K
    c = KV4Cache.allocate(2, 5, 3, 128, "cpu")
    assert c.pages.shape == (2, 5, 3, 2560) and c.n_pages == 5
    with pytest.raises(ValueError, match="16-token"):
        KV4Cache.allocate(2, 5, 3, 128, "cpu", page_size=32)
    with pytest.raises(ValueError, match="64 or 128"):
        K.kv4_page_bytes(80)


@pytest.mark.parametrize("D", [64, 128])
def test_layout_places_every_value_once(D):
    p = plain.places(D)
    seen = np.zeros((20 * D, 2), int)
    for n in "kv":
        at, nib = p[n]
        np.add.at(seen, (at, nib), 1)
    codes = np.r_[0:8 * D, 8 * D + 2 * D:8 * D + 2 * D + 8 * D]
    assert (seen[codes] == 1).all() and seen.sum() == 2 * 16 * D
    for n in "kv":
        starts = np.unique(p[n + "s"])
        assert len(starts) == 16 * D // 32 and starts.max() + p["step"] + 2 <= 20 * D


def test_cpu_tensors_are_refused():
    from fak_b200.ops import kernels as K
    i = lambda *a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        K.kv4_append(torch.zeros(1, 1, 64), torch.zeros(1, 1, 64), i(0), torch.zeros(1, 1, 1280, dtype=torch.uint8))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.kv4_decode_attention(torch.zeros(1, 1, 64), torch.zeros(1, 1, 1280, dtype=torch.uint8), i(0)[None], i(1), torch.zeros(1, 1, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        K.plan_batch(i(0), i(1), i(0)[None], i(1), i(0), 1)
    with pytest.raises(RuntimeError, match="on the GPU"):
        K.token_logprobs(torch.zeros(1, 8), 8, i(0))
