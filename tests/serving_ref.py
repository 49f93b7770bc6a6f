"""Plain 64-bit forms of the serving operators, for the tests (torch on the CPU, loops over requests)."""
import math

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rmsnorm(x, res, gain, eps):
    s = x.double() + (res.double() if res is not None else 0.0)
    return s, s / torch.sqrt(s.pow(2).mean(1, keepdim=True) + eps) * gain.double()


def q8_0(n):
    """(scales f16, codes int) of rows of 32-value blocks, from 64-bit values."""
    b = n.reshape(n.shape[0], -1, 32)
    d = (b.abs().amax(2) / 127.0).float().half()  # the scale passes through fp32, as GGUF's own does
    q = torch.where(d.unsqueeze(2) > 0, torch.round(b / d.double().unsqueeze(2)), torch.zeros_like(b))
    return d, q.clamp(-127, 127).to(torch.int64)


def plan(table, length, new, free, count, bt, ntok, n_blocks):
    """The documented steps, one request at a time, on Python lists."""
    table = [list(r) for r in table]
    free = list(free)
    stack = list(free[:count])
    width = len(table[0]) if table else 0
    nreq = len(length)
    blocks = lambda n: -(-n // bt)
    starts, at = [0], 0
    for r in range(nreq):
        at += max(new[r], 0)
        starts.append(min(at, ntok))
    out_len, kv = list(length), [0] * nreq
    ends = [sum(max(n, 0) for n in new[:r + 1]) for r in range(nreq)]
    for r in range(nreq):
        if new[r] < 0:
            keep = max(length[r] + new[r], 0)
            stack += table[r][blocks(keep):blocks(length[r])]
            out_len[r] = keep
    top = len(stack)
    asked, slots, pos = 0, [-1] * ntok, [-1] * ntok
    pops = 0
    for r in range(nreq):
        kv[r] = out_len[r]
        if new[r] <= 0:
            continue
        have, want = blocks(length[r]), blocks(length[r] + new[r])
        ok = want <= width and ends[r] <= ntok
        if ok:
            asked += want - have
            ok = want == have or asked <= top
        if not ok:
            kv[r] = 0
            continue
        for b in range(have, want):
            table[r][b] = stack[top - 1 - pops]
            pops += 1
        out_len[r] = kv[r] = length[r] + new[r]
        for i in range(new[r]):
            p = length[r] + i
            t = ends[r] - new[r] + i
            pos[t] = p
            pg = table[r][p // bt]
            slots[t] = pg * bt + p % bt if 0 <= pg < n_blocks else -1
    left = top - pops
    for i in range(count, left):
        free[i] = stack[i]
    return table, free, left, out_len, kv, starts, slots, pos


def attention(q, k_cache, v_cache, table, kv_len, q_start, scale, causal=True, window=0):
    """(out, lse, spread): spread[t, h, d] = sum p |v| / sum p, the size rounding errors scale with.
    Only visible keys enter a row's sums, so what it does not see cannot reach it."""
    nt, nh, d = q.shape
    nb, bt, nk, _ = k_cache.shape
    out = torch.zeros(nt, nh, d, dtype=torch.float64)
    spread = torch.zeros_like(out)
    lse = torch.full((nt, nh), -math.inf, dtype=torch.float64)
    smax = 0.0
    for r in range(len(kv_len)):
        n, a, kl = q_start[r + 1] - q_start[r], q_start[r], kv_len[r]
        if n <= 0:
            continue
        keys = torch.arange(kl)
        page = torch.tensor(table[r], dtype=torch.long)[keys // bt] if kl else torch.zeros(0, dtype=torch.long)
        good = (page >= 0) & (page < nb)
        kk = k_cache[page.clamp(0, nb - 1), keys % bt].double() * good.view(-1, 1, 1)
        vv = v_cache[page.clamp(0, nb - 1), keys % bt].double()
        vv = torch.where(good.view(-1, 1, 1), vv, torch.zeros_like(vv))
        kk = torch.where(good.view(-1, 1, 1), kk, torch.zeros_like(kk))
        for i in range(n):
            p = kl - n + i
            hi = min(kl, p + 1) if causal else kl
            lo = max(0, p - window + 1) if window else 0
            if hi <= lo:
                continue
            for h in range(nh):
                g = h // (nh // nk)
                qq = q[a + i, h].double()
                s = scale * (kk[lo:hi, g] @ qq)
                smax = max(smax, scale * float((kk[lo:hi, g].abs() @ qq.abs()).nan_to_num(0, 0, 0).max()))
                m = s.max()
                e = torch.exp(s - m)
                out[a + i, h] = (e @ vv[lo:hi, g]) / e.sum()
                spread[a + i, h] = (e @ vv[lo:hi, g].abs()) / e.sum()
                lse[a + i, h] = m + torch.log(e.sum())
    return out, lse, spread, smax


def attention_bound(out, spread, smax, dim, keys, io, cache):
    """How far a kernel's output may be off.  Scores are sums of dim products in fp32, off by at most
    (dim + 2) 2^-24 of sum |q k| scale; log2 e and the exponential's argument add 4 x 2^-24 of it and
    ex2.approx 2^-22; the weights' sums are at most keys / 8 + 32 additions long, and each output one more
    of that length; 2-byte forms round each weight once; the output is rounded once."""
    u = 2.0 ** -24
    w = 2 * (dim + 6) * u * smax + 2 * 2.0 ** -22 + 2 * (keys / 8 + 32) * u
    if io != torch.float32:
        w += HALF_STEP[cache]
    return w * spread + HALF_STEP[io] * out.abs() + 1e-30
