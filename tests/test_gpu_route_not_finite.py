"""Tokens whose activations are not finite in a routed batch: the exact re-route, which takes them, ends, and the
other tokens' routing is what it is without them."""
import math

import pytest
import torch

from coherence_kernel_b200 import workloads
from coherence_kernel_b200.moe import MoELayer, MoeSpec

pytestmark = pytest.mark.gpu

SPECS = [MoeSpec(1024, 512, 16, 1, 4, 4, 4, 2, 2.5), MoeSpec(1024, 512, 16, 1, 4, 3)]


def layer(spec, ntok, seed=3, router=None):
    w = workloads.make_moe(spec, ntok, seed=seed)
    t = lambda a: torch.from_numpy(a).cuda()
    r = t(w["router"]) if router is None else router(t(w["router"]))
    x = t(w["x"].view("int16")).view(torch.bfloat16)
    return MoELayer(spec, t(w["gate"]), t(w["up"]), t(w["down"]), t(w["s_gate"]), t(w["s_up"]), t(w["s_down"]), r,
                    t(w["bias"]), ntok), x


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("ntok", [8, 200, 600])
def test_tokens_that_are_not_finite(spec, ntok):
    moe, x = layer(spec, ntok)
    _, ids, wts, _ = moe(x)
    bad = x.clone()
    rows = list(range(1, ntok, 2))  # more than 128 of them in the largest batch: the tiled form
    for i, r in enumerate(rows):
        bad[r, (7 * i) % 1024] = [math.nan, math.inf, -math.inf][i % 3]
        if i % 5 == 0:
            bad[r] = math.nan
    out, bids, bwts, counts = moe(bad)
    moe.status(ntok)
    keep = torch.ones(ntok, dtype=torch.bool)
    keep[rows] = False
    assert torch.equal(bids[keep], ids[keep]) and torch.equal(bwts[keep], wts[keep])
    assert torch.isfinite(out[keep]).all()
    valid = (bids >= 0) & (bids < spec.n_experts)
    assert int(counts.sum()) == int(valid.sum())


@pytest.mark.parametrize("spec", SPECS)
@pytest.mark.parametrize("ntok", [1, 8, 300])
def test_no_expert_is_taken_twice(spec, ntok):
    """Two infinite activations whose weights have opposite signs for all experts but two: two scores are numbers."""
    def router(w):
        w = w.view(spec.n_experts, spec.hidden).clone()
        w[:, 5], w[:, 900] = 0.25, -0.25
        w[2, 900] = w[9, 900] = 0.25
        return w
    moe, x = layer(spec, ntok, router=router)
    x[::2, 5] = x[::2, 900] = math.inf
    out, ids, _, counts = moe(x)
    moe.status(ntok)
    for row in ids.tolist():
        real = [e for e in row if 0 <= e < spec.n_experts]
        assert len(set(real)) == len(real)
    assert torch.isfinite(out[1::2]).all() and int(counts.max()) <= ntok
