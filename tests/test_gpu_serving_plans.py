"""Plans of a paged cache at their edges: buffers larger than the step, counts that saturate, padded batches."""
import pytest
import torch

from coherence_kernel_b200 import kv
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def cache(**kw):
    a = dict(n_blocks=16, block_tokens=4, n_heads=4, n_kv_heads=2, head_dim=64, max_requests=3, max_blocks=4, max_tokens=8)
    return kv.PagedKV(**{**a, **kw})


def test_larger_buffers_serve_a_smaller_step():
    """A plan into buffers of an earlier, larger step holds this step's requests and rows only."""
    g = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(8, h, 64, generator=g).cuda() for h in (4, 2, 2))
    got = []
    for larger in (False, True):
        c = cache()
        buf = c.step_buffers(3, 8) if larger else None
        p = c.plan(i32([2, 3, 1]), 8, out=buf)
        c.append(k, v, p)
        c.attend(q, p)
        p = c.plan(i32([1, 1]), 2, out=buf)
        assert [t.numel() for t in (p.length, p.kv_len, p.q_start, p.slots, p.positions)] == [2, 2, 3, 2, 2]
        assert p.length.tolist() == [3, 4] and p.q_start.tolist() == [0, 1, 2]
        with pytest.raises(ValueError):
            c.append(k[:3], v[:3], p)  # the plan has two rows
        c.append(k[6:], v[6:], p)
        out = torch.full_like(q, 77.0)
        c.attend(q, p, out=out)
        assert (out[2:] == 77.0).all()  # no row of the third request, which is not in the step
        got.append((out, c.k.clone(), c.v.clone(), c.length.clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_replaced_buffers_are_checked():
    p = kv.plan_buffers(3, 8, "cuda")
    for name, bad in (("length", torch.empty(4, dtype=torch.int32, device="cuda")), ("slots", i32([0] * 8)),
                      ("kv_len", torch.empty(3, dtype=torch.int64, device="cuda")), ("kv_len", i32([0, 0])),
                      ("q_start", i32([0] * 8)[::2]), ("free_count", i32([])),
                      ("positions", torch.empty(8, dtype=torch.int32))):
        old = getattr(p, name)
        with pytest.raises(ValueError):
            setattr(p, name, bad)
        assert getattr(p, name) is old
    p.length = i32([1, 2])  # fewer requests: the step may have two
    table, free = i32([[-1] * 4] * 3), i32([0, 1, 2, 3])
    with pytest.raises(ValueError):
        kv.plan(table, i32([0, 0, 0]), i32([1, 1, 1]), free, i32([4]), 4, 8, out=p)
    assert kv.plan(table[:2], i32([0, 0]), i32([1, 1]), free, i32([4]), 4, 8, out=p).kv_len.tolist() == [1, 1]


@pytest.mark.parametrize("new", [[2 ** 31 - 1] * 2 + [1], [2 ** 31 - 1] * 4 + [1, 1], [1, 2 ** 30, 2 ** 30, 3], [2 ** 30] * 3,
                                 [3, 2 ** 31 - 1, -2, 2 ** 30, -2 ** 31, 5] * 300])
def test_row_counts_that_saturate(new):
    """No request behind a sum of 2^30 rows or more is served, whatever the sum is."""
    n = len(new)
    table = [[3 * r % (3 * n), 3 * r + 1, -1, -1] for r in range(n)]
    length = [5] * n
    used = {p for row in table for p in row[:2]}
    free = [p for p in range(3 * n) if p not in used]
    free, count = free + [-9] * (3 * n - len(free)), len(free)
    want = ref.plan(table, length, new, free, count, 4, 16, 3 * n)
    t, f = i32(table), i32(free)
    p = kv.plan(t, i32(length), i32(new), f, i32([count]), 4, 16)
    got = (t.tolist(), f.tolist(), int(p.free_count), p.length.tolist(), p.kv_len.tolist(), p.q_start.tolist(),
           p.slots.tolist(), p.positions.tolist())
    for name, a, b in zip(("table", "free", "count", "length", "kv_len", "q_start", "slots", "positions"), got, want):
        assert a == b, name


def test_more_returned_pages_than_the_stack_holds():
    """A count of all pages beside a request that returns three (no consistent state has that): nothing is written
    outside the stack, whose size is the largest."""
    n_blocks = 2 ** 31 - 1
    free = torch.empty(n_blocks, dtype=torch.int32, device="cuda")
    free[-4:] = i32([7, 8, 9, 10])
    table = i32([[1, 2, 3, 4], [-1] * 4])
    p = kv.plan(table, i32([3, 0]), i32([-3, 2]), free, i32([n_blocks]), 1, 4)
    assert p.length.tolist() == [0, 2] and p.kv_len.tolist() == [0, 2] and int(p.free_count) == n_blocks - 2
    assert free[-4:-2].tolist() == [7, 8] and p.positions.tolist() == [0, 1, -1, -1]


def test_windows_past_32_bits_and_negative_ones():
    c = cache(n_heads=4)
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(8, h, 64, generator=g).cuda() for h in (4, 2, 2))
    p = c.plan(i32([8]), 8)
    c.append(k, v, p)
    want = c.attend(q, p)
    for window in (2 ** 31, 2 ** 32 + 1, 10 ** 30):
        assert torch.equal(c.attend(q, p, window=window), want)
    assert not torch.equal(c.attend(q, p, window=1), want)
    with pytest.raises(ValueError):
        c.attend(q, p, window=-1)
