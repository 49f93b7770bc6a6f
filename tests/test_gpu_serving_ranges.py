"""Paged attention where weights and queries span many powers of two: one key far above the rest (an
attention sink), and a query element far above its row's others, over both cache types."""
import math

import pytest
import torch

from tests import serving_ref as ref
from tests.test_gpu_serving import BF16, F16, F32, attn_case, run_attn

pytestmark = pytest.mark.gpu

GAPS = [8.0, 10.0, 12.0, 14.0, 16.0, 17.5, 24.0, 40.0]


def sink_case(gap, jitter, lens, heads, kv_heads, dim, bt, cache, io):
    """Key 0 of every request scores `gap` nats above the others, whose scores differ by about `jitter`; its value is
    zero, so that the small weights are all of the output.  Half of the value columns are 1."""
    q, k, v, table, kl, starts = attn_case(int(gap) + dim, lens, heads, kv_heads, dim, bt, cache, io)
    q, k, v = q / 1.5, k * (jitter / math.sqrt(dim)), v.clone()
    q[..., 0], k[..., 0] = 1.0, 0.0
    v[..., :dim // 2] = 1.0
    for row in table:
        k[row[0], 0], v[row[0], 0] = 0.0, 0.0
        k[row[0], 0, :, 0] = gap
    return q, k, v, table, kl, starts


def check(case, lost=0.0):
    """lost: what a weight of a 16-bit f16 form may lose beside half an ulp, relative to its row's largest weight (it is
    a multiple of f16's smallest subnormal, over the power of two that weights are raised by)."""
    q, k, v, table, kl, starts = case
    out, lse = run_attn(*case, 1.0)
    want, wl, spread, smax = ref.attention(q, k, v, table, kl, starts, 1.0)
    n = max(kl)
    bound = ref.attention_bound(want, spread, smax, q.shape[2], n, q.dtype, k.dtype) + n * lost * float(v.abs().max())
    if q.dtype == F16:
        bound = bound + 2.0 ** -25  # the output's own subnormals
    err = (out.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    lb = 2.0 ** -20 + (2 * (q.shape[2] + 6) * 2.0 ** -24) * smax + (n / 8 + 32) * 2.0 ** -24 + 2.0 ** -23 * wl.abs()
    assert ((lse.double() - wl).abs() <= lb).all()


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("jitter", [0.0, 0.5])
def test_f32_rows_keep_small_weights(gap, cache, jitter):
    check(sink_case(gap, jitter, [(1024, 1), (300, 3), (9, 2)], 2, 1, 64, 16, cache, F32))
    check(sink_case(gap, jitter, [(700, 1)], 3, 3, 128, 16, cache, F32))


@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("dim", [64, 256])
def test_f32_rows_keep_small_query_elements(cache, dim):
    """A query element 2^17 (and 1e36) times the others whose key elements are zero: the scores are those of the rest."""
    for big in (2.0 ** 17, 1e36):
        q, k, v, table, kl, starts = attn_case(dim, [(400, 1), (60, 5)], 4, 2, dim, 16, cache, F32)
        q, k = q.clone(), k.clone()
        q[..., 3], k[..., 3] = big, 0.0
        check((q / 4 if big < 1e30 else q, k, v, table, kl, starts))


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("jitter", [0.0, 0.5])
def test_16_bit_rows_keep_small_weights(gap, cache, jitter):
    lost = 2.0 ** -40 if cache == F16 else 0.0
    check(sink_case(gap, jitter, [(1024, 1), (300, 3), (9, 2)], 2, 1, 64, 16, cache, cache), lost)
    check(sink_case(gap, jitter, [(700, 1)], 3, 3, 128, 16, cache, cache), lost)


@pytest.mark.parametrize("gap", GAPS)
@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("dim,bt", [(64, 16), (128, 12)])
def test_chunks_keep_small_weights(gap, cache, dim, bt):
    lost = 2.0 ** -38 if cache == F16 else 0.0
    check(sink_case(gap, 0.5, [(1100, 100), (90, 90)], 2, 1, dim, bt, cache, cache), lost)
    check(sink_case(gap, 0.0, [(700, 70)], 2, 2, dim, bt, cache, cache), lost)
