"""The serving operators (RMS norm with the residual, KV plan, K/V append, paged attention) against
plain 64-bit forms, at the sizes, masks and layouts where they can go wrong."""
import itertools
import math
import random

import pytest
import torch

from coherence_kernel_b200 import kv, ops
from tests import serving_ref as ref

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g


# ------------------------------------------------------------------------------------------- norm
NORM_BOUND = 50 * 2.0 ** -24  # sums of at most 64 + 12 squares in a chain, halved by the root, and six roundings


@pytest.mark.parametrize("ntok,hidden", [(1, 8), (3, 64), (1, 7168), (5, 1000), (300, 2048), (299, 4104), (301, 8192),
                                         (2, 16384), (297, 16384), (1, 8200)])
@pytest.mark.parametrize("xt,rt,ot", [(F32, F32, BF16), (BF16, F32, F32), (F16, BF16, F16), (BF16, None, BF16)])
def test_norm(ntok, hidden, xt, rt, ot):
    g = gen(ntok * 31 + hidden)
    x = torch.randn(ntok, hidden, generator=g).to(xt)
    res = None if rt is None else (2 * torch.randn(ntok, hidden, generator=g)).to(rt)
    gain = 1 + 0.1 * torch.randn(hidden, generator=g)
    s, n = ref.rmsnorm(x, res, gain, 1e-6)
    rc = None if res is None else res.cuda()
    out = ops.rmsnorm_add(x.cuda(), rc, gain.cuda(), 1e-6, ot).cpu().double()
    assert ((out - n).abs() <= (ref.HALF_STEP[ot] + NORM_BOUND) * n.abs() + (2.0 ** -25 if ot == F16 else 0)).all()
    if res is not None:  # one fp32 addition, then one rounding
        assert torch.equal(rc.cpu(), (x.float() + res.float()).to(rt))


def test_norm_strided_rows_and_separate_sum():
    g = gen(5)
    big = torch.randn(7, 640, generator=g).cuda()
    res = torch.randn(7, 640, generator=g).cuda().to(BF16)
    gain = torch.ones(512).cuda()
    ro = torch.full_like(res, 9.0)
    out = torch.full((7, 520), 5.0, device="cuda")
    ops.rmsnorm_add(big[:, 8:520], res[:, :512], gain, 1e-5, out=out[:, :512], residual_out=ro[:, :512])
    s, n = ref.rmsnorm(big[:, 8:520].cpu(), res[:, :512].cpu(), gain.cpu(), 1e-5)
    assert ((out[:, :512].cpu().double() - n).abs() <= (2.0 ** -24 + NORM_BOUND) * n.abs()).all()
    assert (out[:, 512:] == 5.0).all() and (ro[:, 512:] == 9.0).all()
    assert torch.equal(ro[:, :512].cpu(), s.float().to(BF16))


def q8_parts(blocks, hidden):
    b = blocks.cpu().view(blocks.shape[0], hidden // 32, 34)
    d = b[..., :2].contiguous().view(F16).squeeze(-1)
    return d, b[..., 2:].contiguous().view(torch.int8).to(torch.int64)


@pytest.mark.parametrize("ntok,hidden,xt,rt", [(1, 32, F32, None), (3, 2048, BF16, F32), (300, 2080, F16, BF16),
                                               (2, 7168, F32, F32), (1, 16384, F32, F32), (301, 9216, BF16, F32)])
def test_norm_q8_0_codes_are_the_definitions(ntok, hidden, xt, rt):
    g = gen(hidden)
    x = torch.randn(ntok, hidden, generator=g).to(xt)
    res = None if rt is None else torch.randn(ntok, hidden, generator=g).to(rt)
    gain = 1 + 0.1 * torch.randn(hidden, generator=g)
    if ntok > 1:
        x[1] = 0.0
        if res is not None:
            res[1] = 0.0
        gain[:32] *= 2.0 ** -22  # scales in f16's subnormal range
    _, n = ref.rmsnorm(x, res, gain, float(torch.tensor(1e-6)))
    d, q = ref.q8_0(n)
    blocks = ops.rmsnorm_add(x.cuda(), None if res is None else res.cuda(), gain.cuda(), 1e-6, "q8_0")
    gd, gq = q8_parts(blocks, hidden)
    assert torch.equal(gd.view(torch.int16), d.view(torch.int16))
    assert torch.equal(gq, q)
    values = ops.q8_0_dequant(blocks, 0, ntok * hidden).cpu().view(ntok, -1, 32)
    assert torch.equal(values, d.float().unsqueeze(2) * q.float())


def test_norm_not_finite():
    x = torch.randn(4, 256, generator=gen(1))
    x[1, 7] = math.nan
    x[2, 9] = math.inf
    out = ops.rmsnorm_add(x.cuda(), None, torch.ones(256).cuda(), 1e-6).cpu()
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[3]).all()
    assert torch.isnan(out[1]).all() and torch.isnan(out[2, 9]) and (out[2, :9] == 0).all()
    blocks = ops.rmsnorm_add(x.cuda(), None, torch.ones(256).cuda(), 1e-6, "q8_0")
    v = ops.q8_0_dequant(blocks, 0, 1024).cpu().view(4, 256)
    assert torch.isfinite(v[0]).all() and torch.isfinite(v[3]).all() and torch.isnan(v[1]).all()


# ------------------------------------------------------------------------------------------- plan
def plan_case(seed, nreq, bt, max_len, spare, ntok_slack=5, width_slack=1):
    rng = random.Random(seed)
    length = [rng.choice([0, 1, bt - 1, bt, bt + 1, rng.randrange(0, max_len + 1)]) for _ in range(nreq)]
    new = [rng.choice([0, 1, 1, 1, bt, rng.randrange(0, 2 * bt + 3), -rng.randrange(0, max_len + 1), -1]) for _ in range(nreq)]
    blocks = lambda n: -(-n // bt)
    width = max([max(blocks(l), blocks(max(l + n, 0))) for l, n in zip(length, new)] + [1]) + width_slack
    width = max(width, max([blocks(l) for l in length] + [1]))
    used = sum(blocks(l) for l in length)
    n_blocks = used + spare
    pages = list(range(n_blocks))
    rng.shuffle(pages)
    table = [[-7] * width for _ in range(nreq)]
    at = 0
    for r in range(nreq):
        for b in range(blocks(length[r])):
            table[r][b] = pages[at]
            at += 1
    free = pages[at:] + [-9] * at
    ntok = sum(max(n, 0) for n in new) + ntok_slack
    return table, length, new, free, spare, bt, max(ntok, 0), n_blocks, width


def run_plan(case, alias=False):
    table, length, new, free, count, bt, ntok, n_blocks, width = case
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    t = i(table).view(len(length), width)
    ln, fr, ct = i(length), i(free), i([count])
    out = kv.plan_buffers(len(length), ntok, "cuda")
    if alias:
        out.length, out.free_count = ln, ct
    p = kv.plan(t, ln, i(new), fr, ct, bt, ntok, out=out)
    return (t.tolist(), fr.tolist(), int(p.free_count), p.length.tolist(), p.kv_len.tolist(), p.q_start.tolist(),
            p.slots.tolist(), p.positions.tolist())


@pytest.mark.parametrize("nreq,bt,max_len,spare", [(1, 1, 5, 3), (1, 16, 0, 9), (7, 16, 100, 50), (64, 16, 500, 40),
                                                   (63, 24, 300, 3), (1000, 8, 64, 700), (1025, 128, 300, 5),
                                                   (5000, 16, 90, 2500), (4, 7, 9, 0)])
@pytest.mark.parametrize("alias", [False, True])
def test_plan(nreq, bt, max_len, spare, alias):
    for seed in range(3):
        case = plan_case(seed * 1000 + nreq, nreq, bt, max_len, spare)
        table, length, new, free, count, bt_, ntok, n_blocks, width = case
        want = ref.plan(table, length, new, free, count, bt_, ntok, n_blocks)
        got = run_plan(case, alias)
        for name, a, b in zip(("table", "free", "count", "length", "kv_len", "q_start", "slots", "positions"), got, want):
            assert a == b, name


def test_plan_rows_and_pages_beyond_the_arrays():
    for ntok_slack, width_slack in ((-4, 1), (5, -1), (-30, -2), (3000, 0)):
        for seed in range(4):
            case = plan_case(seed, 20, 8, 60, 40, ntok_slack, width_slack)
            table, length, new, free, count, bt, ntok, n_blocks, width = case
            assert run_plan(case) == ref.plan(table, length, new, free, count, bt, ntok, n_blocks)


def test_plan_long_prompts():
    # more rows and pages than one CTA's threads, and table entries in one request's row
    case = ([[-1] * 9000, [-1] * 9000], [0, 0], [70001, 3], list(range(9999, -1, -1)), 10000, 8, 70016, 10000, 9000)
    assert run_plan(case) == ref.plan(case[0], case[1], case[2], case[3], case[4], 8, 70016, 10000)


def test_plan_no_requests_and_no_rows():
    p = kv.plan(torch.empty((0, 4), dtype=torch.int32, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"),
                torch.empty(0, dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda"),
                torch.tensor([4], dtype=torch.int32, device="cuda"), 16, 3)
    assert p.slots.tolist() == [-1] * 3 and p.q_start.tolist() == [0] and int(p.free_count) == 4


def test_plan_bad_state_stays_inside_the_arrays():
    """Lengths, counts and entries that no consistent state has give slots of -1, never a wild one."""
    i = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    table = i([[3, 99, -5, 2], [0, 1, 2, 3]])
    p = kv.plan(table, i([-4, 2 ** 31 - 1]), i([9, -2 ** 31]), i([77, -1, 5, 2 ** 31 - 1]), i([1000]), 4, 16)
    assert ((p.slots >= -1) & (p.slots < 16)).all()
    p = kv.plan(i([[3, 99, -5, 2]]), i([5]), i([2 ** 31 - 1]), i([0, 1, 2, 3]), i([-3]), 4, 16)
    assert p.slots.tolist() == [-1] * 16 and p.kv_len.tolist() == [0] and p.length.tolist() == [5]
    p = kv.plan(i([[3, 99, -5, 2]]), i([5]), i([2]), i([0, 1, 2, 3]), i([4]), 4, 16)
    assert p.slots.tolist()[:2] == [-1, -1]  # page 99 is outside the cache


# ----------------------------------------------------------------------------------------- append
@pytest.mark.parametrize("ntok,heads,dim,bt", [(1, 1, 8, 1), (5, 3, 72, 7), (64, 8, 128, 16), (1001, 2, 96, 24)])
@pytest.mark.parametrize("xt,ct", [(F32, BF16), (F32, F16), (BF16, BF16), (BF16, F16), (F16, F16)])
def test_append(ntok, heads, dim, bt, xt, ct):
    g = gen(ntok)
    k = (1e3 * torch.randn(ntok, heads, dim, generator=g)).to(xt)
    v = torch.randn(ntok, heads, dim, generator=g).to(xt)
    k[0, 0, 0], v[0, 0, 1], v[0, 0, 2] = math.nan, math.inf, 1e30 if xt != F16 else 6e4
    n_blocks = -(-ntok // bt) + 2
    slots = torch.randperm(n_blocks * bt, generator=g)[:ntok]
    slots[ntok // 2] = -1 if ntok > 1 else slots[0]
    if ntok > 4:
        slots[3] = n_blocks * bt  # just outside
        slots[4] = 2 ** 40
    caches = [torch.full((n_blocks, bt, heads, dim), 3.0).to(ct).cuda() for _ in range(2)]
    kv.append(k.cuda(), v.cuda(), *caches, slots.cuda())
    for rows, cache in zip((k, v), caches):
        want = torch.full((n_blocks * bt, heads, dim), 3.0).to(ct)
        ok = (slots >= 0) & (slots < n_blocks * bt)
        want[slots[ok]] = rows[ok].to(ct)
        got = cache.cpu().view_as(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(got.nan_to_num(0, 7, -7), want.nan_to_num(0, 7, -7))


def test_append_strided_rows_and_head_major_cache():
    g = gen(9)
    qkv = torch.randn(33, 3 * 4 * 64, generator=g).cuda()
    k, v = qkv[:, 256:512].view(33, 4, 64), qkv[:, 512:].view(33, 4, 64)
    kc, vc = (torch.zeros(3, 4, 16, 64, dtype=BF16, device="cuda").permute(0, 2, 1, 3) for _ in range(2))
    slots = torch.arange(33, device="cuda") + 7
    kv.append(k, v, kc, vc, slots)
    flat = kc.reshape(48, 4, 64)
    assert torch.equal(flat[7:40], k.to(BF16)) and (flat[:7] == 0).all()
    assert torch.equal(vc.reshape(48, 4, 64)[7:40], v.to(BF16))


# -------------------------------------------------------------------------------------- attention
def attn_case(seed, lens, heads, kv_heads, dim, bt, cache, io, width_slack=0, head_major=False):
    g = gen(seed)
    blocks = [-(-l // bt) for l, _ in lens]
    n_blocks = sum(blocks) + 2
    shape = (n_blocks, kv_heads, bt, dim) if head_major else (n_blocks, bt, kv_heads, dim)
    mk = lambda: torch.randn(*shape, generator=g).to(cache)
    k, v = mk(), mk()
    if head_major:
        k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
    pages = torch.randperm(n_blocks, generator=g).tolist()
    table = [[-1] * (max(blocks + [1]) + width_slack) for _ in lens]
    at = 0
    for r, nb in enumerate(blocks):
        for b in range(nb):
            table[r][b] = pages[at]
            at += 1
    starts = [0]
    for _, n in lens:
        starts.append(starts[-1] + n)
    q = (1.5 * torch.randn(starts[-1], heads, dim, generator=g)).to(io)
    return q, k, v, table, [l for l, _ in lens], starts


def run_attn(q, k, v, table, kl, starts, scale, pad=0, **kw):
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    nh, d = q.shape[1:]
    at = kv.PagedAttention(nh, k.shape[2], d, q.shape[0] + pad, len(kl))
    qq = torch.cat([q, torch.full((pad, nh, d), math.nan, dtype=q.dtype)]).cuda()
    out = torch.full_like(qq, 77.0)
    lse = torch.full((q.shape[0] + pad, nh), 77.0, device="cuda")
    at(qq, k.cuda(), v.cuda(), i(table), i(kl), i(starts), scale, out=out, lse=lse, **kw)
    at.status()
    assert (out[q.shape[0]:] == 77.0).all() and (lse[q.shape[0]:] == 77.0).all()
    return out[:q.shape[0]].cpu(), lse[:q.shape[0]].cpu()


def check_attn(case, scale=None, pad=0, **kw):
    q, k, v, table, kl, starts = case
    scale = 1 / math.sqrt(q.shape[2]) if scale is None else scale
    out, lse = run_attn(*case, scale, pad, **kw)
    want, wl, spread, smax = ref.attention(q, k, v, table, kl, starts, scale, **kw)
    n = max(kl + [1])
    bound = ref.attention_bound(want, spread, smax, q.shape[2], n, q.dtype, k.dtype)
    err = (out.double() - want).abs()
    assert (err <= bound).all(), float((err / bound).max())
    empty = torch.isinf(wl)
    assert torch.equal(torch.isinf(lse) & (lse < 0), empty) and (out[empty] == 0).all()
    lb = 2.0 ** -20 + (2 * (q.shape[2] + 6) * 2.0 ** -24) * smax + (n / 8 + 32) * 2.0 ** -24 + 2.0 ** -23 * wl[~empty].abs()
    assert ((lse[~empty].double() - wl[~empty]).abs() <= lb).all()


TYPES = [(BF16, BF16), (F16, F16), (BF16, F32), (F16, F32)]


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim", [(1, 1, 64), (8, 2, 128), (5, 1, 80), (6, 6, 8), (4, 2, 256), (20, 1, 96)])
def test_attention_single_tokens(cache, io, heads, kv_heads, dim):
    lens = [(1, 1), (2, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (333, 1), (129, 1)]
    check_attn(attn_case(dim, lens, heads, kv_heads, dim, 16, cache, io), pad=3)


@pytest.mark.parametrize("cache,io", TYPES)
@pytest.mark.parametrize("heads,kv_heads,dim,bt", [(4, 1, 64, 16), (4, 4, 128, 24), (6, 2, 96, 7), (2, 1, 200, 64)])
def test_attention_chunks(cache, io, heads, kv_heads, dim, bt):
    lens = [(40, 40), (100, 1), (77, 13), (130, 65), (5, 0), (64, 64), (200, 17), (1, 1)]
    check_attn(attn_case(bt, lens, heads, kv_heads, dim, bt, cache, io, width_slack=2), pad=5)


CHUNK_LENS = [[(63, 63), (64, 64), (65, 65)], [(200, 127), (300, 128), (129, 129), (2, 1)],
              [(255, 255), (700, 256), (257, 257)], [(1500, 300)], [(0, 0), (900, 40), (5, 5), (400, 150)]]


@pytest.mark.parametrize("lens", CHUNK_LENS)
@pytest.mark.parametrize("cache", [BF16, F16])
@pytest.mark.parametrize("heads,kv_heads,dim,bt", [(2, 2, 128, 16), (1, 1, 64, 24), (3, 1, 96, 128), (2, 1, 8, 1)])
def test_attention_chunk_form(lens, cache, heads, kv_heads, dim, bt):
    check_attn(attn_case(dim + len(lens), lens, heads, kv_heads, dim, bt, cache, cache), pad=2)


@pytest.mark.parametrize("window,causal", [(1, True), (33, True), (200, True), (200, False), (0, False)])
def test_attention_chunk_form_masks(window, causal):
    check_attn(attn_case(window, [(500, 400), (300, 70)], 2, 2, 64, 16, BF16, BF16), causal=causal, window=window)
    case = list(attn_case(3, [(200, 150), (130, 130)], 2, 1, 128, 16, BF16, BF16))
    case[4] = [20, 0]  # most rows before the cache's start; a request that is not served
    check_attn(tuple(case), causal=causal, window=window)


def test_attention_chunk_form_many_heads_over_one():
    check_attn(attn_case(3, [(300, 1), (77, 1), (1, 1), (513, 2)], 128, 1, 128, 16, BF16, BF16))


@pytest.mark.parametrize("group", [1, 3, 4])
def test_attention_chunk_form_head_major_and_odd_groups(group):
    check_attn(attn_case(8, [(270, 150), (333, 90)], 2 * group, 2, 64, 16, BF16, BF16, head_major=True))
    check_attn(attn_case(8, [(270, 150), (333, 90)], 2 * group, 2, 128, 12, F16, F16, head_major=True))


def test_attention_rows_are_independent():
    """A NaN query row reaches no other row, and repeated calls give the same bits."""
    for lens, io in (([(200, 150), (90, 5)], BF16), ([(200, 15), (90, 5)], F32), ([(900, 1)] * 9, BF16)):
        case = attn_case(5, lens, 4, 2, 64, 16, BF16, io)
        clean, _ = run_attn(*case, 0.125)
        q = case[0].clone()
        q[3, 1] = math.nan
        out, _ = run_attn(q, *case[1:], 0.125)
        assert torch.isnan(out[3, 1]).all()
        keep = torch.ones(q.shape[:2], dtype=torch.bool)
        keep[3, 1] = False
        assert torch.equal(out[keep], clean[keep])
        for _ in range(3):
            assert torch.equal(run_attn(*case, 0.125)[0], clean)


def test_attention_on_two_streams_at_once():
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    cases = [attn_case(1, [(700, 300), (90, 1)], 4, 2, 128, 16, BF16, BF16),
             attn_case(2, [(3000, 1)] * 5, 8, 2, 128, 16, BF16, BF16)]
    want = [run_attn(*c, 0.1)[0] for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    objs = [kv.PagedAttention(c[0].shape[1], 2, 128, c[0].shape[0], len(c[4])) for c in cases]
    args = [(c[0].cuda(), c[1].cuda(), c[2].cuda(), i(c[3]), i(c[4]), i(c[5])) for c in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(10):
        for n, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[n].append(objs[n](*args[n], 0.1))
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(x.cpu(), w) for x in o)


def test_cache_past_32_bit_offsets():
    """Pages whose element offsets pass 2^31 and 2^32 bytes: append and both attention forms."""
    n_blocks, bt, kvh, dim = 140000, 16, 8, 128
    big = [torch.zeros((n_blocks, bt, kvh, dim), dtype=BF16, device="cuda") for _ in range(2)]
    g = gen(3)
    lens = [(150, 100), (40, 1)]
    pages = [n_blocks - 1 - 3 * b for b in range(10)] + [131072, 70000, 65537]
    table = [pages[:10], pages[10:] + [0] * 7]
    rows = [torch.randn(190, kvh, dim, generator=g).to(BF16) for _ in range(2)]
    slots = torch.tensor([table[0][p // bt] * bt + p % bt for p in range(150)] +
                         [table[1][p // bt] * bt + p % bt for p in range(40)]).cuda()
    kv.append(rows[0].cuda(), rows[1].cuda(), big[0], big[1], slots)
    small = [torch.zeros((13, bt, kvh, dim), dtype=BF16) for _ in range(2)]
    order = {p: n for n, p in enumerate(pages)}
    for x, r in zip(small, rows):
        for t, s in enumerate(slots.tolist()):
            x[order[s // bt], s % bt] = r[t]
    for x, y in zip(big, small):
        assert torch.equal(x[torch.tensor(pages).cuda()].cpu(), y)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for io in (BF16, F32):
        q = torch.randn(101, 16, dim, generator=g).to(io)
        want, _, spread, smax = ref.attention(q, small[0], small[1], [list(range(10)), [10, 11, 12] + [0] * 7], [150, 40],
                                              [0, 100, 101], 0.1)
        at = kv.PagedAttention(16, kvh, dim, 101, 2)
        out = at(q.cuda(), big[0], big[1], i(table), i([150, 40]), i([0, 100, 101]), 0.1).cpu().double()
        assert ((out - want).abs() <= ref.attention_bound(want, spread, smax, dim, 150, io, BF16)).all()


def test_attention_both_forms_in_one_call():
    """A table wide enough that decode rows and chunks take their own launches (64 or more rows the chunk form)."""
    lens = [(300, 1), (500, 130), (77, 3), (20, 20), (400, 64), (1, 1), (0, 0), (3000, 1)]
    q, k, v, table, kl, starts = attn_case(5, lens, 4, 2, 128, 16, BF16, BF16)
    wide = 8192 * 16 // 16  # 8 requests x 131072 tokens x 2 heads x 128 x 4 bytes: past the one-launch rule
    table = [row + [-1] * (wide - len(row)) for row in table]
    check_attn((q, k, v, table, kl, starts), pad=3)
    check_attn((q, k, v, table, kl, starts), window=100)


def test_attention_chunk_form_growing_scores():
    """Scores that keep growing along the keys: every unit moves the running maximum past the rescaling step."""
    q, k, v, table, kl, starts = attn_case(3, [(1400, 150)], 2, 2, 64, 16, F16, F16)
    order = torch.arange(1400)
    for b, pg in enumerate(table[0]):
        n = min(16, 1400 - b * 16)
        k[pg, :n] = (k[pg, :n] * 0.1 + (order[b * 16:b * 16 + n].view(-1, 1, 1) / 1400)).to(F16)
    q = (q.abs() * 2).to(F16)
    check_attn((q, k, v, table, kl, starts), scale=1.0)
    check_attn((-q, k, v, table, kl, starts), scale=1.0)


@pytest.mark.parametrize("window", [1, 5, 16, 64, 100, 10 ** 9])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_windows_and_no_causal_bound(window, causal):
    lens = [(40, 40), (150, 1), (77, 13), (200, 33)]
    check_attn(attn_case(window % 97, lens, 4, 2, 64, 16, BF16, BF16), causal=causal, window=window)
    check_attn(attn_case(window % 89, lens, 4, 2, 64, 16, BF16, F32), causal=causal, window=window)


def test_attention_rows_that_see_nothing():
    # a request of length 0 with rows (not served), and fewer cached tokens than rows
    case = list(attn_case(3, [(20, 4), (30, 3), (25, 2)], 4, 2, 64, 16, BF16, BF16))
    case[4] = [0, 1, 25]
    check_attn(tuple(case))
    check_attn(tuple(case), causal=False)


@pytest.mark.parametrize("io", [BF16, F32])
def test_attention_head_major_cache(io):
    check_attn(attn_case(8, [(70, 5), (33, 1)], 4, 2, 64, 16, BF16, io, head_major=True))


@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (2, 2, 64)])
def test_attention_long_contexts_split_over_ctas(io, heads, kv_heads, dim):
    check_attn(attn_case(4, [(6000, 1), (2500, 2), (31, 1)], heads, kv_heads, dim, 64, BF16, io))


def test_attention_many_requests():
    rng = random.Random(4)
    lens = [(rng.randrange(1, 60), 1) if r % 7 else (rng.randrange(20, 90), rng.randrange(0, 20)) for r in range(700)]
    check_attn(attn_case(5, lens, 2, 1, 64, 16, BF16, BF16))


def test_attention_chunk_form_takes_nothing_from_what_is_not_seen():
    lens = [(300, 260), (150, 100)]
    q, k, v, table, kl, starts = attn_case(6, lens, 2, 2, 64, 16, BF16, BF16)
    used = {p for r, (l, _) in enumerate(lens) for p in table[r][:-(-l // 16)]}
    for p in range(k.shape[0]):
        if p not in used:
            k[p], v[p] = math.nan, math.inf
    for r, (l, _) in enumerate(lens):
        if l % 16:
            k[table[r][l // 16], l % 16:], v[table[r][l // 16], l % 16:] = math.nan, math.nan
    base = (q, k, v, table, kl, starts)
    check_attn(base)
    clean, _ = run_attn(*base, 0.125)
    for pos, bad in ((30, math.inf), (100, -math.inf), (170, math.nan), (299, math.inf)):
        v2, k2 = v.clone(), k.clone()
        v2[table[0][pos // 16], pos % 16, 1, 5] = bad
        k2[table[1][5], 9, 0, 0] = math.nan  # position 89 of request 1
        out, _ = run_attn(q, k2, v2, table, kl, starts, 0.125)
        first = max(pos - 40, 0)
        other = torch.ones(64, dtype=torch.bool)
        other[5] = False
        assert torch.equal(out[:first], clean[:first])
        hit = out[first:260, 1, 5]
        assert (torch.isnan(hit) if math.isnan(bad) else hit == bad).all()
        assert torch.equal(out[first:260][:, :, other], clean[first:260][:, :, other])
        assert torch.equal(out[:260, 0], clean[:260, 0])
        assert torch.equal(out[260:299], clean[260:299]) and torch.isnan(out[299:, 0]).all()
        assert torch.equal(out[299:, 1], clean[299:, 1])


@pytest.mark.parametrize("io", [BF16, F32])
def test_attention_takes_nothing_from_what_is_not_seen(io):
    """NaN and infinities in unused slots, in other pages, behind the request's end and in later tokens
    of the same chunk do not reach a row; in a visible key or value they do."""
    lens = [(37, 21), (50, 1), (64, 40)]
    q, k, v, table, kl, starts = attn_case(6, lens, 4, 2, 64, 16, BF16, io)
    used = {p for r, (l, _) in enumerate(lens) for p in table[r][:-(-l // 16)]}
    for p in range(k.shape[0]):
        if p not in used:
            k[p], v[p] = math.nan, math.inf
    for r, (l, _) in enumerate(lens):
        if l % 16:
            k[table[r][l // 16], l % 16:], v[table[r][l // 16], l % 16:] = math.nan, math.nan
    base = (q, k, v, table, kl, starts)
    check_attn(base)
    clean, _ = run_attn(*base, 0.125)
    for pos, bad in ((30, math.inf), (36, math.nan)):
        k2, v2 = k.clone(), v.clone()
        v2[table[0][pos // 16], pos % 16, 1, 5] = bad
        k2[table[2][3], 9, 0, 0] = bad  # position 57 of request 2
        out, _ = run_attn(q, k2, v2, table, kl, starts, 0.125)
        first = pos - (37 - 21)
        assert torch.equal(out[:first], clean[:first])
        hit = out[first:21, 2:4, 5]
        assert (torch.isnan(hit) if math.isnan(bad) else hit == bad).all()
        other = torch.ones(64, dtype=torch.bool)
        other[5] = False
        assert torch.equal(out[first:21][:, :, other], clean[first:21][:, :, other])
        assert torch.equal(out[first:21, :2], clean[first:21, :2])
        a = starts[2]
        assert torch.equal(out[a:a + 33], clean[a:a + 33])
        # an infinite key element: the score is infinite by q's sign, so NaN or a weight of zero (f32: NaN)
        want, _, spread, smax = ref.attention(q, k2, v, table, kl, starts, 0.125)
        got, want = out[a + 33:, :2].double(), want[a + 33:, :2]
        nan = torch.isnan(want) | (io == F32)
        assert torch.equal(torch.isnan(got), nan)
        bound = ref.attention_bound(want, spread[a + 33:, :2], smax, 64, 64, io, BF16)
        assert ((got - want).abs() <= bound)[~nan].all()
        assert torch.equal(out[a + 33:, 2:], clean[a + 33:, 2:])


def test_attention_pages_outside_the_cache_read_as_zeros():
    q, k, v, table, kl, starts = attn_case(7, [(60, 3), (50, 1)], 4, 2, 64, 16, BF16, F32)
    table[0][1], table[1][2] = -3, k.shape[0]
    check_attn((q, k, v, table, kl, starts))


def test_attention_lengths_beyond_the_arrays_are_cut():
    q, k, v, table, kl, starts = attn_case(8, [(48, 3), (50, 1)], 4, 2, 64, 16, BF16, F32)
    out, _ = run_attn(q, k, v, table, [10 ** 9, 50], starts, 0.125)
    want, _, _, _ = ref.attention(q, k, v, table, [64, 50], starts, 0.125) if len(table[0]) == 4 else (None,) * 4
    assert torch.allclose(out.double()[:3], want[:3], atol=1e-5)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    at = kv.PagedAttention(4, 2, 64, 4, 2)
    o = at(q.cuda(), k.cuda(), v.cuda(), i(table), i([48, 50]), i([0, 3, 10 ** 9]), 0.125)
    assert torch.isfinite(o).all()


def test_attention_large_scores_and_strided_rows():
    case = attn_case(11, [(300, 9), (77, 1)], 4, 2, 64, 16, F16, F32)
    check_attn((case[0] * 30,) + case[1:])
    q, k, v, table, kl, starts = attn_case(12, [(300, 9), (77, 1)], 4, 2, 64, 16, BF16, BF16)
    wide = torch.zeros(10, 4 * 64 + 128, dtype=BF16, device="cuda")
    qv = wide[:, 64:320].view(10, 4, 64)
    qv.copy_(q)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    at = kv.PagedAttention(4, 2, 64, 10, 2)
    o = at(qv, k.cuda(), v.cuda(), i(table), i(kl), i(starts))
    assert torch.equal(o.cpu(), run_attn(q, k, v, table, kl, starts, 0.125)[0])


# --------------------------------------------------------------------- the operators together
def test_steps_together_and_captured():
    """Prefill, then decode steps through PagedKV: eager and as one replayed graph give the same bits, and
    the last outputs are those of attention over all the K/V rows."""
    def make():
        return kv.PagedKV(n_blocks=64, block_tokens=8, n_heads=4, n_kv_heads=2, head_dim=64, max_requests=3,
                          max_blocks=16, max_tokens=64)
    i = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    g = gen(2)
    prompt, steps = [11, 1, 30], 12
    rows = torch.randn(3, 64 + 3 * steps, 4, 64, generator=g).cuda()
    q_all, k_all, v_all = rows[0], rows[1, :, :2].contiguous(), rows[2, :, :2].contiguous()
    outs = []
    for captured in (False, True):
        c = make()
        p = c.plan(i(prompt), 64)
        c.append(k_all[:64], v_all[:64], p)
        first = c.attend(q_all[:64], p)[:42].clone()
        one, buf = i([1, 1, 1]), c.step_buffers(3, 3)
        qs, ks, vs = q_all[:3].clone(), k_all[:3].clone(), v_all[:3].clone()
        out = torch.empty_like(qs)

        def step():
            pl = c.plan(one, 3, out=buf)
            c.append(ks, vs, pl)
            c.attend(qs, pl, out=out)
        graph = None
        for s in range(steps):
            at = 64 + 3 * s
            qs.copy_(q_all[at:at + 3])
            ks.copy_(k_all[at:at + 3])
            vs.copy_(v_all[at:at + 3])
            if not captured or s == 0:
                step()
            else:
                if graph is None:
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        step()
                graph.replay()
        torch.cuda.synchronize()
        assert c.length.tolist() == [p0 + steps for p0 in prompt]
        outs.append((first, out.clone(), c.table.clone(), c.free_count.clone()))
        # pages come back when requests end
        c.plan(i([-10 ** 6, -5, -10 ** 6]), 3)
        assert c.length.tolist() == [0, 1 + steps - 5, 0] and int(c.free_count) == 63
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    for r in range(3):
        lo = sum(prompt[:r])
        kk = torch.cat([k_all[lo:lo + prompt[r]], k_all[64 + r::3]]).to(BF16).cpu()
        vv = torch.cat([v_all[lo:lo + prompt[r]], v_all[64 + r::3]]).to(BF16).cpu()
        n = kk.shape[0]
        want, _, spread, smax = ref.attention(q_all[64 + 3 * (steps - 1) + r][None].cpu(), kk[None], vv[None], [[0]], [n],
                                              [0, 1], 0.125)
        bound = ref.attention_bound(want, spread, smax, 64, n, F32, BF16)
        assert ((outs[0][1][r].cpu().double() - want[0]).abs() <= bound[0]).all()
