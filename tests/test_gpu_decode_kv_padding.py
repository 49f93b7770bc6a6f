"""The decode step over a paged cache with rows behind the last request: a batch padded to the size a captured step
was recorded for."""
import math

import pytest
import torch

from tests.test_gpu_decode_kv import SPEC, make

pytestmark = pytest.mark.gpu

H, D = SPEC.hidden, 64


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def run(step, mk, kv_heads, new, rows, h0, captured=False):
    """Steps of new[i] tokens per request in batches of rows[i] rows; the last h, and the cache's rows."""
    cache, s = mk(), torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for n, r, x in zip(new, rows, h0):
            plan = cache.plan(i32(n), r)
            h = x[:r].clone()
            q, k, v = (torch.zeros((r, w), device="cuda") for w in (H, kv_heads * D, kv_heads * D))
            if captured:
                keep = h.clone()
                step.run_kv(h, q, k, v, cache, plan)  # loads the kernels
                h.copy_(keep)
                step.capture_kv(h, q, k, v, cache, plan)
                step.replay()
            else:
                step.run_kv(h, q, k, v, cache, plan)
            step.status(r)
    s.synchronize()
    return h, cache


@pytest.mark.parametrize("kv_heads", [16, 4])
@pytest.mark.parametrize("captured", [False, True])
def test_rows_behind_the_last_request_are_left_alone(kv_heads, captured):
    step, *_, mk, rng = make(kv_heads, 16, 5)
    h0 = [torch.from_numpy((rng.standard_normal((16, H)) * 2).astype("float32")).cuda() for _ in range(2)]
    h0[1][4:8] = torch.tensor([1e6, -0.0, math.inf, math.nan], device="cuda").view(4, 1)
    new = ([4, 1, 3], [1, 1, 1])
    h, cache = run(step, mk, kv_heads, new, (16, 8), h0, captured)
    assert torch.equal(h[3:].view(torch.int32), h0[1][3:8].view(torch.int32))  # their own bits
    # the live rows are those of the step without padding
    want, plain = run(step, mk, kv_heads, new, (8, 3), h0)
    assert torch.equal(h[:3], want)
    assert torch.equal(cache.k, plain.k) and torch.equal(cache.v, plain.v)


def test_no_request_and_nobody_served():
    """No request: every row is padding.  A request without pages: its rows attend over nothing, and count as rows."""
    step, *_, mk, rng = make(4, 8, 6)
    h0 = torch.from_numpy((rng.standard_normal((8, H)) * 2).astype("float32")).cuda()
    h, cache = run(step, mk, 4, [[]], [8], [h0])
    assert torch.equal(h, h0) and (cache.k == 0).all()
    h, cache = run(step, mk, 4, [[0, 0, 0]], [8], [h0])
    assert torch.equal(h, h0) and (cache.k == 0).all()
    a, cache = run(step, mk, 4, [[1000, 2, 0]], [8], [h0])  # 1000 rows do not fit
    assert (cache.k == 0).all() and not torch.equal(a, h0)


def test_windows_of_the_step():
    step, *_, mk, rng = make(4, 8, 6)
    cache = mk()
    plan = cache.plan(i32([3, 2, 1]), 6)
    f = lambda w: torch.zeros((6, w), device="cuda")
    with pytest.raises(ValueError):
        step.run_kv(f(H), f(H), f(4 * D), f(4 * D), cache, plan, window=-1)
    h0, hs = torch.from_numpy(rng.standard_normal((6, H)).astype("float32")).cuda(), []
    for window in (0, 2 ** 32 + 1, 1):
        h = h0.clone()
        step.run_kv(h, f(H), f(4 * D), f(4 * D), cache, plan, window=window)
        hs.append(h)
    assert torch.equal(hs[0], hs[1]) and not torch.equal(hs[0], hs[2])


def test_a_captured_step_holds_its_buffers():
    """Buffers that only the captured step still refers to are not handed out again."""
    step, *_, mk, rng = make(4, 8, 6)
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        cache = mk()
        plan = cache.plan(i32([1, 1, 1]), 3, out=cache.step_buffers(3, 3))
        h, q, k, v = (torch.zeros((3, w), device="cuda") for w in (H, H, 4 * D, 4 * D))
        step.run_kv(h, q, k, v, cache, plan)
        step.capture_kv(h, q, k, v, cache, plan)
        step.replay()
        sizes = [t.shape for t in (h, q, k, v, cache.attention.ws, cache.k, cache.v)]
        s.synchronize()
        del h, q, k, v, cache, plan
        mine = [torch.full(z, 77.0, device="cuda", dtype=d) for z in sizes for d in (torch.float32, torch.uint8, torch.bfloat16)]
        step.replay()
    s.synchronize()
    assert all((t == 77).all() for t in mine)
