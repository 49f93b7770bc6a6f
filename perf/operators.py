"""The serving operators around the KV cache, as measured cases.

Four operators of one forward pass over a batch of requests: the RMS norm with the residual's
addition ("norm"), the block tables and slot maps of a paged KV cache ("plan"), the write of new
K/V rows through the slot map ("append") and the attention of each request's new tokens over its
cached ones ("attn").  `run` computes them in plain torch operations, or with this package's
kernels when `own` is set.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token through the FFN norm of a decode step at the DeepSeek-V3 hidden size: latency
        dict(name="norm_step_1", op="norm", ntok=1, hidden=7168, x="f32", res="f32", out="bf16"),
        # a medium batch of the 2048-wide model, output in 8-bit blocks with scales
        dict(name="norm_q8_509", op="norm", ntok=509, hidden=2048, x="bf16", res="f32", out="q8_0"),
        # the 8192-token prefill batch of the benchmark's layer, MoE output added to the f32 stream
        dict(name="norm_prefill_8192", op="norm", ntok=8192, hidden=7168, x="bf16", res="f32", out="bf16"),
        # a decode step of 64 requests: one new token each, a page boundary here and there
        dict(name="plan_step_64", op="plan", nreq=64, max_len=8192, block=16, mode="step", scarce=False),
        # a busy scheduler tick: 1000 requests, some finish, some roll back, some get prompt chunks
        dict(name="plan_mixed_1000", op="plan", nreq=1000, max_len=4096, block=16, mode="mixed", scarce=False),
        # the K/V rows of a 64-request decode step (f32 projections) into a bf16 cache
        dict(name="append_step_64", op="append", ntok=64, heads=8, dim=128, block=16, x="f32", cache="bf16"),
        # the K/V rows of an 8192-token prefill batch
        dict(name="append_prefill_8192", op="append", ntok=8192, heads=8, dim=128, block=16, x="bf16", cache="bf16"),
        # the decode step's own form: one request, every projection row a head of its own, f32 activations
        dict(name="attn_step_1", op="attn", heads=56, kv_heads=56, dim=128, block=16, io="f32", cache="bf16",
             window=0, lse=False, nreq=1, max_new=1, max_ctx=1000, ragged=False),
        # a decode batch of 64 ragged requests with grouped heads
        dict(name="attn_decode_64", op="attn", heads=32, kv_heads=8, dim=128, block=16, io="bf16", cache="bf16",
             window=0, lse=False, nreq=64, max_new=1, max_ctx=8192, ragged=True),
        # one request with a very long context, log-sum-exp kept for joining with another cache's part
        dict(name="attn_decode_131072", op="attn", heads=32, kv_heads=8, dim=128, block=64, io="f16", cache="f16",
             window=0, lse=True, nreq=1, max_new=1, max_ctx=131072, ragged=False),
        # chunked prefill: 2048 new tokens at the end of 8192
        dict(name="attn_chunk_2048", op="attn", heads=32, kv_heads=8, dim=128, block=16, io="bf16", cache="bf16",
             window=0, lse=False, nreq=1, max_new=2048, max_ctx=8192, ragged=False),
        # a ragged mix of decode rows and odd chunks, odd page size, smaller heads, sliding window
        dict(name="attn_mixed_17", op="attn", heads=16, kv_heads=4, dim=96, block=24, io="bf16", cache="bf16",
             window=1000, lse=False, nreq=17, max_new=333, max_ctx=5000, ragged=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "plan", "append", "attn", "attn"])
    if op == "norm":
        return dict(op=op, ntok=_log_int(rng, 1, 8192), hidden=32 * _log_int(rng, 2, 224), x=rng.choice(list(_TYPES)),
                    res=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16", "f16", "q8_0"]))
    if op == "plan":
        return dict(op=op, nreq=_log_int(rng, 1, 1000), max_len=_log_int(rng, 64, 4096),
                    block=rng.choice([1, 8, 16, 24, 64, 128]), mode=rng.choice(["step", "mixed"]),
                    scarce=rng.random() < 0.3)
    if op == "append":
        cache = rng.choice(["bf16", "f16"])
        return dict(op=op, ntok=_log_int(rng, 1, 8192), heads=rng.choice([1, 2, 4, 8]), dim=rng.choice([64, 96, 128]),
                    block=rng.choice([8, 16, 24, 64]), x=rng.choice(["f32", cache]), cache=cache)
    cache = rng.choice(["bf16", "f16"])
    kvh = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    case = dict(op=op, heads=kvh * min(group, 32 // kvh), kv_heads=kvh, dim=rng.choice([64, 80, 96, 128]),
                block=rng.choice([8, 16, 24, 64, 128]), io=cache, cache=cache, window=rng.choice([0, 0, 0, 100, 1024]),
                lse=rng.random() < 0.5, ragged=rng.random() < 0.7)
    kind = rng.choice(["decode", "long", "chunk", "mixed"])
    if kind == "decode":
        case.update(nreq=_log_int(rng, 1, 64), max_new=1, max_ctx=_log_int(rng, 1, 8192), io=rng.choice(["f32", cache]))
    elif kind == "long":
        case.update(nreq=1, max_new=1, max_ctx=_log_int(rng, 8192, 131072))
    elif kind == "chunk":
        n = _log_int(rng, 16, 2048)
        case.update(nreq=1, max_new=n, max_ctx=n + rng.randrange(0, 8193 - n))
    else:
        case.update(nreq=rng.randrange(2, 20), max_new=_log_int(rng, 2, 333), max_ctx=_log_int(rng, 400, 5000),
                    io=rng.choice(["f32", cache]))
    return case


# -------------------------------------------------------------------- lengths and tables (host side)
def _host_rng(case, seed):
    import random
    return random.Random(f"{sorted((k, v) for k, v in case.items() if k != 'name')}/{seed}")


def _attn_lengths(case):
    """(cached + new, new) of every request: fixed by the case, so that work() is the case's own."""
    rng = _host_rng(case, "lengths")
    out = []
    for r in range(case["nreq"]):
        if not case["ragged"]:
            out.append((case["max_ctx"], case["max_new"]))
            continue
        new = 1 if (case["max_new"] == 1 or r % 3 == 0) else rng.randrange(1, case["max_new"] + 1)
        out.append((max(new, rng.randrange(1, case["max_ctx"] + 1)), new))
    return out


def _plan_lengths(case):
    rng = _host_rng(case, "lengths")
    out = []
    for r in range(case["nreq"]):
        ln = rng.randrange(1, case["max_len"] + 1)
        if case["mode"] == "step":
            out.append((ln, 1))
        else:
            kind = rng.random()
            if kind < 0.5:
                out.append((ln, 1))                                     # decodes
            elif kind < 0.6:
                out.append((ln, -ln))                                   # finished
            elif kind < 0.7:
                out.append((ln, -rng.randrange(0, min(ln, 8) + 1)))     # rejected drafts
            elif kind < 0.9:
                out.append((0, rng.randrange(1, 257)))                  # new prompt
            else:
                out.append((ln, rng.randrange(0, 65)))                  # next chunk
    return out


def _cdiv(a, b):
    return -(-a // b)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)
    st = dict(case=case)
    if case["op"] == "norm":
        n, h = case["ntok"], case["hidden"]
        st["x"] = normal(n, h).to(_TYPES[case["x"]])
        st["res"] = (2 * normal(n, h)).to(_TYPES[case["res"]])
        st["gain"] = 1 + 0.1 * normal(h)
        st["res_out"] = torch.empty_like(st["res"])
        st["eps"] = 1e-6
        return st
    if case["op"] == "plan":
        b = case["block"]
        lens = _plan_lengths(case)
        blocks = [_cdiv(max(ln, ln + new), b) for ln, new in lens]
        width = max(blocks) + 1
        used = sum(_cdiv(ln, b) for ln, _ in lens)
        # scarce: pages for about half of the growth, so that the last requests are not served
        total = used + (sum(blocks) - used) // 2 + 1 if case["scarce"] else sum(blocks) + 16
        perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        have = torch.tensor([_cdiv(ln, b) for ln, _ in lens], device=dev)
        first = torch.cumsum(have, 0) - have
        col = torch.arange(width, device=dev)
        held = col[None, :] < have[:, None]
        src = (first[:, None] + col[None, :]).clamp(max=total - 1)
        st["table"] = torch.where(held, perm[src], torch.full_like(perm[src], -1))
        st["free"] = torch.full((total,), -1, dtype=torch.int32, device=dev)
        st["free"][: total - used] = perm[used:]
        st["free_count"] = torch.tensor([total - used], dtype=torch.int32, device=dev)
        st["len"] = torch.tensor([ln for ln, _ in lens], dtype=torch.int32, device=dev)
        st["new"] = torch.tensor([new for _, new in lens], dtype=torch.int32, device=dev)
        # rows are padded to a multiple of 64, as a program that captures its step per batch size pads them
        st["ntok"] = max(64, _cdiv(sum(max(n, 0) for _, n in lens), 64) * 64)
        st["n_blocks"] = total
        if own:
            from coherence_kernel_b200 import kv
            st["outs"] = kv.plan_buffers(case["nreq"], st["ntok"], dev)
        return st
    if case["op"] == "append":
        n, h, d, b = case["ntok"], case["heads"], case["dim"], case["block"]
        st["k"] = normal(n, h, d).to(_TYPES[case["x"]])
        st["v"] = normal(n, h, d).to(_TYPES[case["x"]])
        blocks = _cdiv(n, b) + 3
        st["k_cache"] = torch.zeros((blocks, b, h, d), dtype=_TYPES[case["cache"]], device=dev)
        st["v_cache"] = torch.zeros_like(st["k_cache"])
        # requests' rows run through their pages in order; every seventh row is padding
        page = torch.randperm(blocks, generator=g, device=dev)
        t = torch.arange(n, device=dev)
        slot = page[t // b] * b + t % b
        st["slots"] = torch.where(t % 7 == 6, torch.full_like(slot, -1), slot)
        return st
    lens = _attn_lengths(case)
    b, hk, d = case["block"], case["kv_heads"], case["dim"]
    blocks = [_cdiv(ln, b) for ln, _ in lens]
    total = sum(blocks) + 1
    cache_t = _TYPES[case["cache"]]
    st["k_cache"] = normal(total, b, hk, d).to(cache_t)
    st["v_cache"] = normal(total, b, hk, d).to(cache_t)
    perm = torch.randperm(total, generator=g, device=dev).to(torch.int32)
    table = torch.zeros((len(lens), max(blocks)), dtype=torch.int32, device=dev)
    at = 0
    for r, nb in enumerate(blocks):
        table[r, :nb] = perm[at:at + nb]
        at += nb
    st["table"] = table
    st["lens"] = lens
    starts = [0]
    for _, new in lens:
        starts.append(starts[-1] + new)
    st["starts"] = starts
    st["kv_len"] = torch.tensor([ln for ln, _ in lens], dtype=torch.int32, device=dev)
    st["q_start"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    st["q"] = normal(starts[-1], case["heads"], d).to(_TYPES[case["io"]])
    st["scale"] = 1.0 / math.sqrt(d)
    if own:
        from coherence_kernel_b200 import kv
        st["attend"] = kv.PagedAttention(case["heads"], hk, d, max_tokens=starts[-1], max_requests=len(lens),
                                         device=dev)
    return st


# ----------------------------------------------------------------------------------- the plain forms
def _q8_0_values(n):
    """What Q8_0 blocks of n hold: per 32 values a half-precision scale and codes in -127..127."""
    v = n.reshape(-1, 32)
    d = (v.abs().amax(1, keepdim=True) / 127).half().to(v.dtype)
    q = torch.where(d > 0, torch.round(v / d).clamp(-127, 127), torch.zeros_like(v))
    return (q * d).float().reshape(n.shape)


def _plain_norm(st):
    case = st["case"]
    # a code flips where a value lies next to the border of two, so the 8-bit form is taken in 64 bits
    f = torch.float64 if case["out"] == "q8_0" else torch.float32
    s = st["x"].to(f) + st["res"].to(f)
    n = s * (1.0 / torch.sqrt((s * s).mean(1, keepdim=True) + st["eps"])) * st["gain"].to(f)
    out = _q8_0_values(n) if case["out"] == "q8_0" else n.to(_TYPES[case["out"]])
    return out, s.to(_TYPES[case["res"]])


def _plain_plan(st):
    b, ntok = st["case"]["block"], st["ntok"]
    ln, new, table = st["len"].long(), st["new"].long(), st["table"].long()
    free, count = st["free"].long(), st["free_count"].long()
    dev = ln.device
    nreq, width = table.shape
    rows = new.clamp(min=0)
    after = (ln + new).clamp(min=0)
    have, want = (ln + b - 1) // b, (after + b - 1) // b
    row_end = torch.cumsum(rows, 0)
    fits = (rows > 0) & (want <= width) & (row_end <= ntok)
    need = torch.where(fits, want - have, torch.zeros_like(want))
    back = torch.where(new < 0, have - want, torch.zeros_like(want))
    col = torch.arange(width, device=dev)[None, :]
    # the stack with the returned blocks pushed: request by request, in block order
    back_end = torch.cumsum(back, 0)
    returned = (col >= want[:, None]) & (col < (want + back)[:, None])
    at = count + (back_end - back)[:, None] + col - want[:, None]
    size = free.numel()
    stack = torch.cat([free, free.new_zeros(1)])
    stack = stack.scatter(0, torch.where(returned, at, torch.full_like(at, size)).reshape(-1), table.reshape(-1))
    top = count + back_end[-1]
    need_end = torch.cumsum(need, 0)
    served = fits & ((need == 0) | (need_end <= top))
    taken = torch.where(served, need, torch.zeros_like(need))
    fresh = (col >= have[:, None]) & (col < (have + taken)[:, None])
    k = top - 1 - ((need_end - need)[:, None] + col - have[:, None])
    table_out = torch.where(fresh, stack[k.clamp(0, size)], table)
    count_out = top - taken.sum()
    idx = torch.arange(size, device=dev)
    free_out = torch.where((idx >= count) & (idx < count_out), stack[:size], free)
    grows = new >= 0
    len_out = torch.where(grows & ~served, ln, after)
    kv_len = torch.where((rows > 0) & ~served, torch.zeros_like(ln), len_out)
    q_start = torch.cat([row_end.new_zeros(1), row_end]).clamp(max=ntok)
    t = torch.arange(ntok, device=dev)
    r = torch.searchsorted(row_end, t, right=True).clamp(max=nreq - 1)
    live = (t < q_start[-1]) & served[r]
    pos = ln[r] + t - (row_end - rows)[r]
    page = table_out[r, (pos // b).clamp(0, width - 1)]
    slot = torch.where(live, page * b + pos % b, torch.full_like(pos, -1))
    pos = torch.where(live, pos, torch.full_like(pos, -1))
    i32 = torch.int32
    return (table_out.to(i32), free_out.to(i32), count_out.to(i32).reshape(1), len_out.to(i32), kv_len.to(i32),
            q_start.to(i32), slot, pos.to(i32))


def _plain_append(st):
    keep = st["slots"] >= 0
    where = st["slots"][keep]
    outs = []
    for rows, cache in ((st["k"], st["k_cache"]), (st["v"], st["v_cache"])):
        flat = cache.view(-1, cache.shape[2], cache.shape[3])
        flat[where] = rows[keep].to(cache.dtype)
        outs.append(cache)
    return tuple(outs)


def _visible(n_new, n_keys, lo, window, dev):
    """Which of the keys lo .. n_keys - 1 each of the last n_new tokens of a request sees."""
    i = torch.arange(n_keys - n_new, n_keys, device=dev)[:, None]
    j = torch.arange(lo, n_keys, device=dev)[None, :]
    see = j <= i
    if window:
        see = see & (j > i - window)
    return see


def _plain_attn(st):
    case = st["case"]
    dev = st["q"].device
    b, hk, d, win = case["block"], case["kv_heads"], case["dim"], case["window"]
    grp = case["heads"] // hk
    out = torch.empty_like(st["q"])
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float32, device=dev) if case["lse"] else None
    kf, vf = st["k_cache"].view(-1, hk, d), st["v_cache"].view(-1, hk, d)
    for r, (ln, new) in enumerate(st["lens"]):
        t0 = st["starts"][r]
        lo = max(0, ln - new - win + 1) if win else 0
        j = torch.arange(lo, ln, device=dev)
        idx = st["table"][r][j // b].long() * b + j % b
        hide = ~_visible(new, ln, lo, win, dev) if (new > 1 or win) else None
        for h in range(hk) if new > 64 else [slice(0, hk)]:
            h = slice(h, h + 1) if isinstance(h, int) else h
            k = kf[idx][:, h].float().permute(1, 2, 0)                     # [heads, d, keys]
            v = vf[idx][:, h].float().permute(1, 0, 2)
            qh = slice(h.start * grp, h.stop * grp)
            q = st["q"][t0:t0 + new, qh].float().reshape(new, -1, grp, d).permute(1, 2, 0, 3)
            n = q.shape[0]
            s = torch.matmul(q.reshape(n, grp * new, d), k) * st["scale"]
            if hide is not None:
                s = s.view(n, grp, new, -1).masked_fill_(hide, float("-inf")).view(n, grp * new, -1)
            m = s.amax(2, keepdim=True)
            p = torch.exp(s - m)
            z = p.sum(2, keepdim=True)
            o = torch.matmul(p, v) / z
            out[t0:t0 + new, qh] = o.view(n, grp, new, d).permute(2, 0, 1, 3).reshape(new, -1, d).to(out.dtype)
            if lse is not None:
                lse[t0:t0 + new, qh] = (m + torch.log(z)).view(n, grp, new).permute(2, 0, 1).reshape(new, -1)
    return (out, lse) if lse is not None else (out,)


# ------------------------------------------------------------------------------ the framework's calls
def _own_norm(st):
    from coherence_kernel_b200 import ops
    case = st["case"]
    n, h = case["ntok"], case["hidden"]
    if case["out"] == "q8_0":
        blocks = ops.rmsnorm_add(st["x"], st["res"], st["gain"], st["eps"], "q8_0", residual_out=st["res_out"])
        return ops.q8_0_dequant(blocks, 0, n * h).view(n, h), st["res_out"]
    out = ops.rmsnorm_add(st["x"], st["res"], st["gain"], st["eps"], _TYPES[case["out"]], residual_out=st["res_out"])
    return out, st["res_out"]


def _own_plan(st):
    from coherence_kernel_b200 import kv
    p = kv.plan(st["table"], st["len"], st["new"], st["free"], st["free_count"], st["case"]["block"], st["ntok"],
                out=st["outs"])
    return st["table"], st["free"], p.free_count, p.length, p.kv_len, p.q_start, p.slots, p.positions


def _own_append(st):
    from coherence_kernel_b200 import kv
    kv.append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["slots"])
    return st["k_cache"], st["v_cache"]


def _own_attn(st):
    case = st["case"]
    r = st["attend"](st["q"], st["k_cache"], st["v_cache"], st["table"], st["kv_len"], st["q_start"], st["scale"],
                     window=case["window"], return_lse=case["lse"])
    return r if case["lse"] else (r,)


def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "plan": _own_plan, "append": _own_append, "attn": _own_attn}[op](state)
    return {"norm": _plain_norm, "plan": _plain_plan, "append": _plain_append, "attn": _plain_attn}[op](state)


# ------------------------------------------------------------------------------------ the bare needs
def _pairs(ln, new, window):
    """Visible (query, key) pairs of the last `new` tokens of ln."""
    total = 0
    for i in range(ln - new, ln):
        total += min(i + 1, window) if window else i + 1
    return total


def work(case):
    size = {"f32": 4, "bf16": 2, "f16": 2, "q8_0": 34 / 32}
    if case["op"] == "norm":
        n = case["ntok"] * case["hidden"]
        return {"bytes": int(n * (size[case["x"]] + 2 * size[case["res"]] + size[case["out"]]) + 4 * case["hidden"]),
                "flops": 6 * n}
    if case["op"] == "plan":
        b = case["block"]
        lens = _plan_lengths(case)
        ntok = max(64, _cdiv(sum(max(n, 0) for _, n in lens), 64) * 64)
        moved = sum(abs(_cdiv(max(ln + n, 0), b) - _cdiv(ln, b)) for ln, n in lens)
        return {"bytes": 20 * len(lens) + 12 * ntok + 8 * moved, "flops": 4 * ntok}
    if case["op"] == "append":
        n = case["ntok"] * case["heads"] * case["dim"]
        live = case["ntok"] - case["ntok"] // 7
        n = n * live // case["ntok"]
        return {"bytes": 2 * n * (size[case["x"]] + size[case["cache"]]) + 8 * case["ntok"], "flops": 2 * n}
    hk, d, h = case["kv_heads"], case["dim"], case["heads"]
    lens = _attn_lengths(case)
    win = case["window"]
    keys = sum(ln - max(0, ln - new - win + 1) if win else ln for ln, new in lens)
    rows = sum(new for _, new in lens)
    pairs = sum(_pairs(ln, new, win) for ln, new in lens)
    by = 2 * keys * hk * d * 2 + 2 * rows * h * d * size[case["io"]] + (4 * rows * h if case["lse"] else 0)
    return {"bytes": int(by), "flops": 4 * d * h * pairs}


# --------------------------------------------------------------------------- the definition, 64 bits
def _host_attn_rows(q, k, v, scale, first, window, lo):
    """Attention of the rows q [n, d] (row i at position first + i) over k, v (rows lo ..), in 64 bits."""
    s = scale * (q @ k.T)
    n, m = s.shape
    pos = first + torch.arange(n, device=q.device).view(n, 1)
    key = lo + torch.arange(m, device=q.device).view(1, m)
    gone = key > pos
    if window:
        gone |= key <= pos - window
    s[gone] = -float("inf")
    top = s.max(dim=1).values
    e = torch.exp(s - top.view(n, 1))
    z = e.sum(dim=1)
    return (e @ v) / z.view(n, 1), top + torch.log(z)


def exact(case, seed):
    if case["op"] in ("plan", "append"):
        return None
    st = prepare(case, seed)
    if case["op"] == "norm":
        x, r, g = st["x"].double(), st["res"].double(), st["gain"].double()
        s = x + r
        y = g * s / torch.sqrt(s.pow(2).sum(1, keepdim=True) / case["hidden"] + st["eps"])
        if case["out"] == "q8_0":
            blk = y.reshape(case["ntok"], -1, 32)
            d = torch.max(blk.abs(), dim=2, keepdim=True).values.div(127).half().double()
            q = torch.nan_to_num(blk / d).round().clamp(min=-127, max=127)
            y = (d * q).reshape(case["ntok"], -1)
        return y, s
    if work(case)["flops"] > 4e11:
        return None
    b, hk, d, win = case["block"], case["kv_heads"], case["dim"], case["window"]
    grp = case["heads"] // hk
    q = st["q"].double()
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], dtype=torch.float64, device=q.device)
    for r, (ln, new) in enumerate(st["lens"]):
        lo = max(0, ln - new - win + 1) if win else 0
        first_page, last_page = lo // b, _cdiv(ln, b)
        pages = st["table"][r, first_page:last_page].long()
        kk = st["k_cache"][pages].flatten(0, 1)[lo - first_page * b:ln - first_page * b]
        vv = st["v_cache"][pages].flatten(0, 1)[lo - first_page * b:ln - first_page * b]
        t0 = st["starts"][r]
        for h in range(case["heads"]):
            k1, v1 = kk[:, h // grp].double(), vv[:, h // grp].double()
            o, z = _host_attn_rows(q[t0:t0 + new, h], k1, v1, st["scale"], ln - new, win, lo)
            out[t0:t0 + new, h] = o
            lse[t0:t0 + new, h] = z
    return (out, lse) if case["lse"] else (out,)
