"""The decode step over a paged KV cache (DecodeStep.run_kv): a prefill of several requests and decode
steps, each stage against the oracle and the plain attention on the step's own intermediates, and the
captured step, with a plan before each replay, against the eager one."""
import numpy as np
import pytest
import torch

from coherence_kernel_b200 import kv, synth, workloads
from coherence_kernel_b200.decode import DecodeStep
from coherence_kernel_b200.moe import MoeSpec
from oracle import oracle as O
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

SPEC = MoeSpec(1024, 512, 16, 1, 4, 4, 4, 2, 2.5)


def make(kv_heads, T, seed):
    H, D = SPEC.hidden, 64
    rng = np.random.default_rng(seed)
    w = workloads.make_moe(SPEC, T, seed=seed)
    t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
    rows = [H, kv_heads * D, kv_heads * D, H]
    dense = [synth.make_q4k(np.random.default_rng([seed, i]), r * H) for i, r in enumerate(rows)]
    g = [(1 + 0.1 * rng.standard_normal(H)).astype(np.float32) for _ in range(2)]
    step = DecodeStep(SPEC, *[t(d) for d in dense], t(g[0]), t(g[1]), t(w["gate"]), t(w["up"]), t(w["down"]),
                      t(w["s_gate"]), t(w["s_up"]), t(w["s_down"]), t(w["router"]), t(w["bias"]), max_tokens=T,
                      kv_rows=kv_heads * D)
    mk = lambda: kv.PagedKV(n_blocks=24, block_tokens=8, n_heads=H // D, n_kv_heads=kv_heads, head_dim=D,
                            max_requests=3, max_blocks=6, max_tokens=T)
    return step, w, dense, g, mk, rng


def dot(q4, rows, x):
    m = O.q4k_dequant(q4, 0, rows * x.shape[1]).reshape(rows, x.shape[1])
    return x.astype(np.float64) @ m.T, np.abs(x.astype(np.float64)) @ np.abs(m).T


@pytest.mark.parametrize("kv_heads", [16, 4])
def test_step_over_the_cache_matches_the_oracle(kv_heads):
    T, H, D = 32, SPEC.hidden, 64
    step, w, dense, g, mk, rng = make(kv_heads, T, 5)
    cache, R = mk(), kv_heads * D
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for new in ([9, 1, 14], [1, 1, 1], [1, 3, 0], [1, 1, 1]):
        n = sum(new)
        plan = cache.plan(i32(new), n)
        h0 = (rng.standard_normal((n, H)) * 2).astype(np.float32)
        h = torch.from_numpy(h0).cuda()
        q, k, v = (torch.empty((n, r), device="cuda") for r in (H, R, R))
        step.run_kv(h, q, k, v, cache, plan)
        step.status(n)
        vw = {a: b.clone() for a, b in step.views(n).items()}
        a = np.stack([O.rmsnorm(x.astype(np.float64), g[0].astype(np.float64), 1e-6) for x in h0])
        for out, m, r in ((q, dense[0], H), (k, dense[1], R), (v, dense[2], R)):
            want, bound = dot(m, r, a)
            assert np.all(np.abs(out.cpu().numpy() - want) <= 1e-3 * bound)
        # the cache holds this step's rows, rounded once
        s = plan.slots
        for rows, c in ((k, cache.k), (v, cache.v)):
            assert torch.equal(c.view(-1, kv_heads, D)[s], rows.view(n, kv_heads, D).to(torch.bfloat16))
        kl, starts, table = plan.kv_len.tolist(), plan.q_start.tolist(), cache.table.tolist()
        want, _, spread, smax = ref.attention(q.view(n, H // D, D).cpu(), cache.k.cpu(), cache.v.cpu(), table, kl, starts,
                                              D ** -0.5)
        got = vw["a"].view(n, H // D, D).cpu().double()  # the attention's output
        assert ((got - want).abs() <= ref.attention_bound(want, spread, smax, D, max(kl), torch.float32,
                                                          torch.bfloat16)).all()
        want, bound = dot(dense[3], H, vw["a"].cpu().numpy())
        assert np.all(np.abs(vw["o"].cpu().numpy() - want) <= 1e-3 * bound)
        h1 = h0 + vw["o"].cpu().numpy()
        b = vw["b"].view(torch.int16).cpu().numpy().view(np.uint16)
        nb = np.stack([O.rmsnorm(x.astype(np.float64), g[1].astype(np.float64), 1e-6) for x in h1])
        assert np.all(np.abs(synth.bf16_bits_to_f32(b) - nb) <= (2.0 ** -8 + 2.0 ** -18) * np.abs(nb))
        cfg = O.moe_cfg(SPEC.hidden, SPEC.inter, SPEC.n_experts, SPEC.n_shared, SPEC.nsel, SPEC.mode, SPEC.ngroups,
                        SPEC.topk_groups, SPEC.wscale)
        rids, _, rout = O.moe_layer(cfg, w, np.ascontiguousarray(b), np.arange(n))
        assert np.array_equal(vw["ids"].cpu().numpy(), rids)
        m = vw["m"].float().cpu().numpy()
        for t in range(n):
            assert np.abs(m[t] - rout[t]).max() <= 2e-2 * np.abs(rout[t]).max()
        assert np.array_equal(h.cpu().numpy(), h1 + m)


def test_captured_step_with_a_plan_before_each_replay():
    T, H, D, kvh = 8, SPEC.hidden, 64, 4
    step, w, dense, g, mk, rng = make(kvh, T, 6)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    hs = [torch.from_numpy((rng.standard_normal((3, H)) * 2).astype(np.float32)).cuda() for _ in range(20)]
    results = []
    s = torch.cuda.Stream()
    for captured in (False, True):
        cache, one, got = mk(), i32([1, 1, 1]), []
        buf = cache.step_buffers(3, 3)
        h, q, k, v = torch.empty((3, H), device="cuda"), *(torch.empty((3, r), device="cuda") for r in (H, kvh * D, kvh * D))
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            for i, h0 in enumerate(hs):
                h.copy_(h0)
                cache.plan(one, 3, out=buf)
                if captured and i == 0:
                    step.run_kv(h, q, k, v, cache, buf)  # loads the kernels; the capture records the same call
                    step.capture_kv(h, q, k, v, cache, buf)
                elif captured:
                    step.replay()
                else:
                    step.run_kv(h, q, k, v, cache, buf)
                got.append(h.clone())
            step.status(3)
        torch.cuda.synchronize()
        assert cache.length.tolist() == [20, 20, 20]
        results.append((got, cache.k.clone(), cache.v.clone()))
    for a, b in zip(results[0][0], results[1][0]):
        assert torch.equal(a, b)
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])


def test_step_kv_refusals():
    step, w, dense, g, mk, rng = make(4, 8, 7)
    cache = mk()
    plan = cache.plan(torch.tensor([1, 1, 1], dtype=torch.int32, device="cuda"), 3)
    f = lambda n, r: torch.empty((n, r), device="cuda")
    with pytest.raises(ValueError):
        step.run(f(3, 1024), f(3, 1024), f(3, 1024), f(3, 1024))     # grouped heads need a cache
    with pytest.raises(ValueError):
        step.run_kv(f(4, 1024), f(4, 1024), f(4, 256), f(4, 256), cache, plan)  # more rows than the plan
    other = kv.PagedKV(8, 8, 16, 8, 64, 3, 4, 8)
    with pytest.raises(ValueError):
        step.run_kv(f(3, 1024), f(3, 1024), f(3, 256), f(3, 256), other, plan)  # other heads
    with pytest.raises(ValueError):
        step.run_kv(f(9, 1024), f(9, 1024), f(9, 256), f(9, 256), cache, plan)
