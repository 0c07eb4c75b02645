"""The batch plan built on the GPU against a plain loop over requests and tokens."""
import numpy as np
import pytest
import torch

import kv4_plain as plain

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def make(old, new, seed=0, width=None, spare=5):
    rng = np.random.RandomState(seed)
    have, need = [-(-a // 16) for a in old], [-(-(a + n) // 16) for a, n in zip(old, new)]
    ids = rng.permutation(sum(need) + spare + 1).astype(np.int32)
    table = np.zeros((len(old), width or max(need + [1])), np.int32)
    at = 0
    for b, h in enumerate(have):
        table[b, :h] = ids[at:at + h]
        at += h
    return table, ids[at:]


def dev(x):
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


CASES = [([0], [1]), ([0, 0], [0, 0]), ([15, 16, 17, 0], [1, 1, 1, 1]), ([5, 0, 40], [0, 100, 3]),
         (list(range(0, 600, 2)), [i % 23 for i in range(300)]), ([100] * 1500, [1] * 1500), ([0], [5000])]


@pytest.mark.parametrize("old,new", CASES)
@pytest.mark.parametrize("slack,held", [(0, False), (7, True)])
def test_plan(K, old, new, slack, held):
    table, free = make(old, new, seed=len(old))
    cap, head = sum(new) + slack, 2 if slack else 0
    free = np.concatenate([np.full(head, 99999, np.int32), free])
    t = dev(table)
    out = K.BatchPlan.allocate(len(old), cap, "cuda") if held else None
    p = K.plan_batch(dev(old), dev(new), t, dev(free), dev([head]), cap, out)
    want = plain.plan(old, new, table, free, head, cap)
    for name, w in want.items():
        np.testing.assert_array_equal(getattr(p, name).cpu().numpy(), w, err_msg=name)
    np.testing.assert_array_equal(t.cpu().numpy(), table)
    if held:
        assert p.slot.data_ptr() == out.slot.data_ptr()


def test_plan_of_no_requests(K):
    p = K.plan_batch(dev([]), dev([]), torch.zeros(0, 4, dtype=torch.int32, device="cuda"), dev([1, 2]), dev([1]), 3)
    assert p.slot.tolist() == [-1, -1, -1] and p.q_off.tolist() == [0] and p.free_head.tolist() == [1]


@pytest.mark.parametrize("kind", ["pages", "table", "tokens", "negative"])
def test_plan_reports_what_does_not_fit(K, kind):
    err = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.register_error_word(err.device, err)
    try:
        old, new = [10, 0], [10, 40]
        table, free = make(old, new, width=4)
        cap = 50
        if kind == "pages":
            free = free[:2]
        if kind == "table":
            table = table[:, :2].copy()
        if kind == "tokens":
            cap = 30
        if kind == "negative":
            new = [-3, 40]
        t = dev(table)
        p = K.plan_batch(dev(old), dev(new), t, dev(free), dev([0]), cap)
        assert err.item() == 2
        slot = p.slot.cpu().numpy()
        if kind == "pages":       # the third page is missing: positions 16 .. 39 of request 1
            assert (slot[:26] >= 0).all() and (slot[26:] == -1).all()
        if kind == "table":       # positions 32 .. 39 of request 1
            assert (slot[:42] >= 0).all() and (slot[42:] == -1).all()
        if kind == "tokens":
            assert p.q_off.tolist() == [0, 10, 30] and p.last.tolist() == [9, -1] and (slot >= 0).all()
        if kind == "negative":
            assert p.q_off.tolist() == [0, 0, 40] and p.ctx.tolist() == [10, 40]
    finally:
        K.register_error_word(err.device, None)


def test_plan_in_a_graph_follows_the_lengths(K):
    old, new, head = dev([16, 3]), dev([1, 1]), dev([0])
    t, free = dev([[7, 0, 0], [8, 0, 0]]), dev([1, 2, 3, 4])
    plan = K.BatchPlan.allocate(2, 2, "cuda")
    K.plan_batch(old, new, t, free, head, 2, plan)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        K.plan_batch(old, new, t, free, head, 2, plan)
        old.copy_(plan.ctx)
        head.copy_(plan.free_head)
    old.copy_(dev([16, 3]))
    head.zero_()
    g.replay()
    assert plan.slot.tolist() == [1 * 16, 8 * 16 + 3] and head.tolist() == [1]
    for _ in range(12):
        g.replay()
    g.replay()      # position 17 + 12 = 29 and 16
    assert plan.pos.tolist() == [29, 16] and plan.slot.tolist() == [16 + 13, 2 * 16] and head.tolist() == [2]


def test_refusals(K):
    with pytest.raises(RuntimeError, match="CUDA"):
        K.plan_batch(torch.zeros(1, dtype=torch.int32), dev([1]), dev([[0]]), dev([1]), dev([0]), 1)
    with pytest.raises(RuntimeError, match="new ones"):
        K.plan_batch(dev([1, 2]), dev([1]), dev([[0], [0]]), dev([1]), dev([0]), 1)
    with pytest.raises(RuntimeError, match="block table"):
        K.plan_batch(dev([1, 2]), dev([1, 1]), dev([[0]]), dev([1]), dev([0]), 2)
    with pytest.raises(RuntimeError, match="int32"):
        K.plan_batch(dev([1]).long(), dev([1]), dev([[0]]), dev([1]), dev([0]), 1)
    with pytest.raises(RuntimeError, match="word of its own"):
        h = dev([0])
        K.plan_batch(dev([1]), dev([1]), dev([[0]]), dev([1]), h, 1, K.BatchPlan.allocate(1, 1, "cuda")._replace(free_head=h))
