"""Refusals of the serving entry points, checked on the host: each is answered before any device work."""
import ctypes

import pytest

from coherence_kernel_b200 import _lib

P = 0x10000  # a non-null, aligned address that no refused call reads
ESHAPE, EARG = -2, -3


def norm(L, **kw):
    a = dict(xt=0, x=P, xs=256, rt=0, res=P, ro=P, rs=256, gain=P, ot=30, out=P, os=256, ntok=4, hidden=256, eps=1e-6)
    a.update(kw)
    return L.ck_rmsnorm_add(a["xt"], a["x"], a["xs"], a["rt"], a["res"], a["ro"], a["rs"], a["gain"], a["ot"], a["out"],
                            a["os"], a["ntok"], a["hidden"], a["eps"], None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), EARG), (dict(gain=None), EARG), (dict(out=None), EARG), (dict(res=None), EARG), (dict(xt=8), EARG),
    (dict(rt=12), EARG), (dict(ot=12), EARG), (dict(hidden=0), ESHAPE), (dict(hidden=252), ESHAPE),
    (dict(hidden=16392, xs=16392, rs=16392, os=16392), ESHAPE), (dict(hidden=248, ot=8), ESHAPE), (dict(x=P + 8), EARG),
    (dict(out=P + 2), EARG), (dict(out=P + 1, ot=8), EARG), (dict(xs=255), EARG), (dict(xs=260), EARG),
    (dict(rs=128), EARG), (dict(os=128), EARG)])
def test_norm_refusals(cuda_lib, kw, rc):
    assert norm(cuda_lib, **kw) == rc
    assert b"ck_rmsnorm_add" in cuda_lib.ck_last_error()


def test_norm_no_rows(cuda_lib):
    assert norm(cuda_lib, ntok=0, x=None, out=None) == 0


def plan(L, **kw):
    a = dict(ln=P, new=P, nreq=4, table=P, ts=8, mb=8, free=P, ci=P, nb=64, bt=16, ntok=32, lo=P, co=P, kl=P, qs=P, sl=P,
             pos=P)
    a.update(kw)
    return L.ck_kv_plan(a["ln"], a["new"], a["nreq"], a["table"], a["ts"], a["mb"], a["free"], a["ci"], a["nb"], a["bt"],
                        a["ntok"], a["lo"], a["co"], a["kl"], a["qs"], a["sl"], a["pos"], None)


@pytest.mark.parametrize("kw,rc", [
    (dict(ln=None), EARG), (dict(new=None), EARG), (dict(table=None), EARG), (dict(free=None), EARG),
    (dict(ci=None), EARG), (dict(lo=None), EARG), (dict(co=None), EARG), (dict(kl=None), EARG), (dict(qs=None), EARG),
    (dict(sl=None), EARG), (dict(pos=None), EARG), (dict(ts=7), EARG), (dict(nreq=8193), ESHAPE),
    (dict(ntok=1 << 30), ESHAPE), (dict(bt=0), ESHAPE), (dict(mb=0, ts=0), ESHAPE), (dict(nb=0), ESHAPE),
    (dict(mb=1 << 27, ts=1 << 27), ESHAPE), (dict(nb=1 << 27), ESHAPE)])
def test_plan_refusals(cuda_lib, kw, rc):
    assert plan(cuda_lib, **kw) == rc
    assert b"ck_kv_plan" in cuda_lib.ck_last_error()


CFG = dict(h=2, d=64, bt=16, nb=64, t=30, sb=2048, st=128, sh=64)


def config(**kw):
    c = {**CFG, **kw}
    return _lib.KvConfig(c["h"], c["d"], c["bt"], c["nb"], c["t"], 0, c["sb"], c["st"], c["sh"])


BAD_CONFIGS = [(dict(h=0), ESHAPE), (dict(d=0), ESHAPE), (dict(d=60), ESHAPE), (dict(d=264), ESHAPE), (dict(bt=0), ESHAPE),
               (dict(nb=0), ESHAPE), (dict(nb=1 << 27), ESHAPE), (dict(t=0), EARG), (dict(t=8), EARG), (dict(sb=2047), EARG),
               (dict(st=4), EARG), (dict(sh=1), EARG)]


def append(L, cfg=None, **kw):
    a = dict(t=0, k=P, ks=128, v=P, vs=128, sl=P, ntok=4, kc=P, vc=P)
    a.update(kw)
    return L.ck_kv_append(ctypes.byref(cfg if cfg is not None else config()), a["t"], a["k"], a["ks"], a["v"], a["vs"],
                          a["sl"], a["ntok"], a["kc"], a["vc"], None)


@pytest.mark.parametrize("kw,rc", BAD_CONFIGS)
def test_append_bad_configs(cuda_lib, kw, rc):
    assert append(cuda_lib, config(**kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(t=12), EARG), (dict(k=None), EARG), (dict(v=P + 4), EARG), (dict(sl=None), EARG), (dict(kc=P + 8), EARG),
    (dict(vc=None), EARG), (dict(ks=120), EARG), (dict(vs=132), EARG), (dict(ntok=1 << 25), ESHAPE)])
def test_append_refusals(cuda_lib, kw, rc):
    assert append(cuda_lib, **kw) == rc
    assert append(cuda_lib, ntok=0, k=None) == 0


def attend(L, cfg=None, **kw):
    a = dict(nh=4, t=30, q=P, qs=256, kc=P, vc=P, table=P, ts=8, mb=8, kl=P, st=P, nreq=2, ntok=4, scale=0.1, causal=1,
             window=0, out=P, os=256, lse=None, ws=P, wsb=None)
    a.update(kw)
    wsb = L.ck_paged_attention_workspace_bytes(4, 2, 64) if a["wsb"] is None else a["wsb"]
    return L.ck_paged_attention(ctypes.byref(cfg if cfg is not None else config()), a["nh"], a["t"], a["q"], a["qs"],
                                a["kc"], a["vc"], a["table"], a["ts"], a["mb"], a["kl"], a["st"], a["nreq"], a["ntok"],
                                a["scale"], a["causal"], a["window"], a["out"], a["os"], a["lse"], a["ws"], wsb, None)


@pytest.mark.parametrize("kw,rc", BAD_CONFIGS)
def test_attention_bad_configs(cuda_lib, kw, rc):
    assert attend(cuda_lib, config(**kw)) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(nh=0), ESHAPE), (dict(nh=3), ESHAPE), (dict(t=1), EARG), (dict(t=8), EARG), (dict(q=None), EARG),
    (dict(q=P + 8), EARG), (dict(out=P + 2), EARG), (dict(kc=None), EARG), (dict(vc=P + 1), EARG), (dict(table=None), EARG),
    (dict(kl=None), EARG), (dict(st=None), EARG), (dict(ws=None), EARG), (dict(wsb=16), EARG), (dict(qs=248), EARG),
    (dict(os=260), EARG), (dict(ts=4), EARG), (dict(mb=0), ESHAPE), (dict(mb=1 << 27, ts=1 << 27), ESHAPE),
    (dict(ntok=1 << 28), ESHAPE), (dict(scale=0.0), EARG), (dict(scale=-1.0), EARG),
    (dict(scale=float("nan")), EARG), (dict(scale=float("inf")), EARG)])
def test_attention_refusals(cuda_lib, kw, rc):
    assert attend(cuda_lib, **kw) == rc
    assert b"ck_paged_attention" in cuda_lib.ck_last_error()


def test_attention_nothing_to_do(cuda_lib):
    assert attend(cuda_lib, ntok=0, q=None) == 0 and attend(cuda_lib, nreq=0, q=None) == 0


def test_attention_workspace_refuses_bad_heads(cuda_lib):
    f = cuda_lib.ck_paged_attention_workspace_bytes
    assert f(8, 2, 128) > 0 and f(8, 3, 128) == 0 and f(8, 2, 100) == 0 and f(0, 1, 64) == 0 and f(8, 2, 264) == 0
