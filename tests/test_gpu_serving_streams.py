"""A cache and its attention made on one stream and used on another."""
import torch
import pytest

from coherence_kernel_b200 import kv
from tests.test_gpu_serving import BF16, attn_case, run_attn

pytestmark = pytest.mark.gpu


def test_made_on_a_busy_stream_and_used_on_another():
    """The workspace's counts and the cache's pages are zero when the constructor returns, whatever the stream still does."""
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    case = attn_case(1, [(5000, 1), (900, 1)], 8, 2, 64, 16, BF16, BF16)
    want = run_attn(*case, 0.1)[0]
    q, k, v, table, kl, starts = case
    args = [q.cuda(), k.cuda(), v.cuda(), i(table), i(kl), i(starts)]
    at = kv.PagedAttention(8, 2, 64, 2, 2)
    dirty = [torch.full((at.ws_bytes,), 1, dtype=torch.uint8, device="cuda") for _ in range(4)]
    cache_bytes = 64 * 16 * 2 * 64
    dirty += [torch.full((cache_bytes,), 7.0, dtype=BF16, device="cuda") for _ in range(4)]
    torch.cuda.synchronize()
    del dirty  # the next allocations of these sizes are not zero
    side = torch.cuda.Stream()
    torch.cuda._sleep(100_000_000)  # some 50 ms of the current stream
    at = kv.PagedAttention(8, 2, 64, 2, 2)
    with torch.cuda.stream(side):
        out = at(*args, 0.1)
    side.synchronize()
    assert torch.equal(out.cpu(), want)
    torch.cuda._sleep(100_000_000)
    cache = kv.PagedKV(64, 16, 8, 2, 64, max_requests=2, max_blocks=8, max_tokens=4)
    with torch.cuda.stream(side):
        p = cache.plan(i([2, 1]).clone(), 4)
        rows = torch.ones((4, 2, 64), device="cuda")
        cache.append(rows, rows, p)
    side.synchronize()
    torch.cuda.synchronize()
    assert cache.length.tolist() == [2, 1] and int(cache.free_count) == 62
    assert int((cache.k != 0).sum()) == 3 * 2 * 64
