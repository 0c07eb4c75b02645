"""The batch plan where it can go wrong: plans in the memory of their own inputs, pages past 32-bit slots."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def K():
    from fak_b200.ops import kernels
    return kernels


def dev(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("which", ["cached", "new", "free pages", "table", "one another", "inside"])
def test_a_plan_in_its_inputs_memory_is_refused(K, which):
    """Other CTAs still read the lengths when the first writes the plan, and it reads them again itself."""
    p = K.BatchPlan.allocate(3, 8, "cuda")
    a = {"cached": dev([1, 2, 3]), "new": dev([1, 1, 1]), "block_table": torch.zeros(3, 4, dtype=torch.int32, device="cuda"),
         "free_pages": dev([5, 6, 7]), "free_head": dev([0])}
    if which == "cached":
        a["cached"] = p.ctx
    elif which == "new":
        a["new"] = p.last
    elif which == "free pages":
        a["free_pages"] = p.seq[2:]
    elif which == "table":
        p = p._replace(slot=a["block_table"].view(-1)[3:11])
    elif which == "one another":
        p = p._replace(pos=p.slot)
    else:       # the last row of the table ends where the offsets begin
        buf = torch.zeros(64, dtype=torch.int32, device="cuda")
        a["block_table"] = buf[:60].view(3, 20)[:, :4]
        p = p._replace(q_off=buf[43:47])
    with pytest.raises(RuntimeError, match="memory"):
        K.plan_batch(*a.values(), 8, p)


def test_a_plan_between_the_rows_of_its_table(K):
    """Memory that nothing else touches may lie anywhere, and vectors may be longer than the plan."""
    buf = torch.zeros(60, dtype=torch.int32, device="cuda")
    table = buf.view(3, 20)[:, :4]
    p = K.BatchPlan.allocate(3, 8, "cuda")._replace(q_off=buf[4:17], ctx=buf[17:24], slot=buf[24:32], last=buf[44:47])
    table[:, 0] = dev([4, 5, 6])
    r = K.plan_batch(dev([1, 2, 16]), dev([1, 2, 1]), table, dev([9]), dev([0]), 8, p)
    assert r.q_off[:4].tolist() == [0, 1, 3, 4] and r.ctx[:3].tolist() == [2, 4, 17] and r.last.tolist() == [0, 2, 3]
    assert r.slot.tolist() == [65, 82, 83, 144, -1, -1, -1, -1] and table.tolist() == [[4, 0, 0, 0], [5, 0, 0, 0], [6, 9, 0, 0]]


@pytest.fixture
def err(K):
    word = torch.zeros(1, dtype=torch.int32, device="cuda")
    K.register_error_word(word.device, word)
    yield word
    K.register_error_word(word.device, None)


@pytest.mark.parametrize("where", ["table", "free pages"])
def test_pages_at_the_end_of_32_bit_slots(K, err, where):
    last = (2 ** 31 - 1) // 16
    for page, slots, code in ((last, [2 ** 31 - 15], 0), (last + 1, [-1], 2), (2 ** 28, [-1], 2), (-1, [-1], 2)):
        err.zero_()
        if where == "table":
            p = K.plan_batch(dev([1]), dev([1]), dev([[page]]), dev([0]), dev([0]), 1)
        else:
            p = K.plan_batch(dev([0]), dev([2]), dev([[0]]), dev([page]), dev([0]), 2)
            slots = [slots[0] - 1 if slots[0] > 0 else -1, slots[0]]
        assert p.slot.tolist() == slots and err.item() == code


@pytest.mark.parametrize("new", [[2 ** 31 - 1, 2 ** 31 - 1], [3] + [2 ** 30] * 4 + [5], [2 ** 30] * 600, [1, 2 ** 31 - 1, 1, 1]])
def test_tokens_past_32_bits_are_reported(K, err, new):
    """Sums that would come back to a small or negative number are tokens past the capacity like others."""
    B, cap = len(new), 16
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None].contiguous()
    p = K.plan_batch(dev([0] * B), dev(new), table, dev(list(range(B))), dev([0]), cap)
    assert err.item() == 2
    want = [0]
    for n in new:
        want.append(min(cap, want[-1] + n))
    assert p.q_off.tolist() == want and p.ctx.tolist() == new
    assert p.last.tolist() == [sum(new[:b + 1]) - 1 if sum(new[:b + 1]) <= cap else -1 for b in range(B)]
    assert p.seq.tolist() == [next(b for b in range(B) if i < sum(new[:b + 1])) for i in range(cap)]


def test_a_plan_is_saved(K, tmp_path):
    p = K.plan_batch(dev([1]), dev([2]), dev([[3]]), dev([4]), dev([0]), 4)
    torch.save(tuple(p), tmp_path / "p.pt")
    assert all(torch.equal(a, b) for a, b in zip(p, torch.load(tmp_path / "p.pt")))
