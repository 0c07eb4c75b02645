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
