"""What the language-model operators refuse: the C ABI checks its arguments
before any CUDA call, so this runs without a GPU."""
import ctypes

import pytest
import torch

import vxb

P = 0x1000  # a 16-byte aligned address that is never read: every call here is refused, or has no rows


def rc(name, *args):
    return getattr(vxb.lib(), "vxb_" + name)(*args)


NORM = dict(type=vxb.TYPE_BF16, N=4, C=256, x=P, xs=256, res=None, rs=0, sum=None, ss=0, wt=vxb.TYPE_BF16, w=P,
            eps=1e-6, yt=vxb.TYPE_E4M3, y=P, ys=256, scale=P, scs=2, st=None)


@pytest.mark.parametrize("change", [
    dict(type=vxb.TYPE_Q4_0), dict(type=7), dict(wt=vxb.TYPE_F16), dict(yt=vxb.TYPE_F16), dict(N=-1), dict(C=0),
    dict(C=32769, xs=40000, ys=40000, scs=400), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")),
    dict(x=None), dict(w=None), dict(y=None), dict(scale=None), dict(yt=vxb.TYPE_BF16), dict(xs=255), dict(ys=255),
    dict(scs=1), dict(res=P, rs=100), dict(sum=P, ss=255), dict(x=P + 1), dict(scale=P + 2)])
def test_rms_norm_refuses(change):
    a = {**NORM, **change}
    assert rc("rms_norm", *a.values()) == vxb.ERR_INVALID_ARGUMENT
    assert b"rms_norm" in vxb.lib().vxb_last_error()


def test_no_rows_is_a_success_without_work():
    assert rc("rms_norm", *{**NORM, "N": 0}.values()) == vxb.OK
    assert rc("fp8_product", *{**PROD, "N": 0}.values()) == vxb.OK
    assert rc("rotary", *{**ROT, "N": 0}.values()) == vxb.OK
    assert rc("rotary_append", *{**APPEND, "N": 0}.values()) == vxb.OK
    assert rc("paged_attention", *{**ATTN, "N": 0}.values()) == vxb.OK
    assert rc("paged_attention", *{**ATTN, "B": 0}.values()) == vxb.OK


PROD = dict(N=4, K=256, M=100, x=P, xs=256, sc=P, scs=2, w=P, ws=256, wsc=P, bias=None, yt=vxb.TYPE_F16, y=P, ys=100,
            st=None)


@pytest.mark.parametrize("change", [
    dict(N=-1), dict(K=0), dict(K=250), dict(K=8), dict(M=0), dict(yt=vxb.TYPE_E4M3), dict(yt=vxb.TYPE_Q4_0),
    dict(x=None), dict(sc=None), dict(w=None), dict(wsc=None), dict(y=None), dict(xs=240), dict(ws=240), dict(ys=99),
    dict(scs=1), dict(x=P + 8), dict(w=P + 4), dict(xs=264), dict(ws=264), dict(y=P + 1), dict(bias=P + 1),
    dict(N=2 ** 31)])
def test_fp8_product_refuses(change):
    assert rc("fp8_product", *{**PROD, **change}.values()) == vxb.ERR_INVALID_ARGUMENT


ROT = dict(type=vxb.TYPE_F16, N=4, Hq=4, Hk=2, D=64, R=64, inter=0, factor=1.0, pos=P, freq=P, q=P, qt=256, qh=64,
           qo=P, qot=256, qoh=64, k=P, kt=128, kh=64, ko=P, kot=128, koh=64, st=None)


@pytest.mark.parametrize("change", [
    dict(type=vxb.TYPE_E4M3), dict(N=-1), dict(Hq=0), dict(D=0), dict(R=0), dict(R=63), dict(R=66), dict(D=512, R=258),
    dict(factor=float("nan")), dict(factor=float("inf")), dict(pos=None), dict(freq=None), dict(q=None), dict(qo=None),
    dict(k=None), dict(ko=None), dict(Hk=0), dict(q=P + 1), dict(pos=P + 4), dict(D=2000)])
def test_rotary_refuses(change):
    assert rc("rotary", *{**ROT, **change}.values()) == vxb.ERR_INVALID_ARGUMENT


APPEND = dict(type=vxb.TYPE_F16, N=4, Hq=4, Hk=2, D=64, R=64, inter=0, factor=1.0, pos=P, slots=P, freq=P, q=P, qt=256,
              qh=64, qo=P, qot=256, qoh=64, k=P, kt=128, kh=64, v=P, vt=128, vh=64, kc=P, vc=P, pages=8, page=16,
              ps=2048, ss=128, hs=64, st=None)


@pytest.mark.parametrize("change", [
    dict(slots=None), dict(k=None), dict(v=None), dict(kc=None), dict(vc=None), dict(pages=-1), dict(page=0),
    dict(Hk=0), dict(R=7), dict(slots=P + 4), dict(vc=P + 1), dict(pages=2 ** 62)])
def test_rotary_append_refuses(change):
    assert rc("rotary_append", *{**APPEND, **change}.values()) == vxb.ERR_INVALID_ARGUMENT


ATTN = dict(type=vxb.TYPE_BF16, N=4, B=2, Hq=8, Hk=2, D=64, q=P, qt=512, qh=64, kc=P, vc=P, pages=8, page=16, ps=2048,
            ss=128, hs=64, table=P, ts=4, mp=4, cu=P, kv=P, scale=0.125, window=0, out=P, ot=512, oh=64, wsp=None,
            wsb=0, st=None)


@pytest.mark.parametrize("change", [
    dict(type=vxb.TYPE_F32), dict(type=vxb.TYPE_E4M3), dict(N=-1), dict(B=-1), dict(Hq=7), dict(Hk=0), dict(D=60),
    dict(D=136), dict(D=0), dict(page=8), dict(page=24), dict(page=0), dict(pages=-1), dict(mp=-1),
    dict(mp=2 ** 27, ts=2 ** 27), dict(mp=2 ** 26, ts=2 ** 26), dict(N=2 ** 30 + 1), dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None),
    dict(out=None), dict(kc=None), dict(vc=None), dict(table=None), dict(cu=None), dict(kv=None), dict(ts=3),
    dict(q=P + 8), dict(kc=P + 2), dict(qt=513), dict(qh=60), dict(ps=2049), dict(ss=129), dict(hs=63),
    dict(out=P + 1), dict(table=P + 2)])
def test_paged_attention_refuses(change):
    assert rc("paged_attention", *{**ATTN, **change}.values()) == vxb.ERR_INVALID_ARGUMENT


def test_workspace_refuses_what_the_call_refuses():
    assert vxb.lib().vxb_paged_attention_workspace(4, 2, 7, 2, 64, 4, 16) == -1
    assert vxb.lib().vxb_paged_attention_workspace(4, 2, 8, 2, 60, 4, 16) == -1
    assert b"paged_attention" in vxb.lib().vxb_last_error()


def refused(f, *args, **kw):
    with pytest.raises(vxb.VxbError) as e:
        f(*args, **kw)
    assert e.value.code == vxb.ERR_INVALID_ARGUMENT


def test_wrappers_refuse_tensors_off_the_gpu_and_of_wrong_form():
    bf, f8 = torch.bfloat16, torch.float8_e4m3fn
    x, w, y = torch.zeros(4, 256, dtype=bf), torch.zeros(256, dtype=bf), torch.zeros(4, 256, dtype=bf)
    refused(vxb.rms_norm, x, w, y)  # not on a CUDA device
    refused(vxb.rms_norm, x, w[:128], y)
    refused(vxb.rms_norm, x.t(), w[:4], y.t())
    refused(vxb.rms_norm, x, w, y, residual=x.half())
    refused(vxb.rms_norm, x, w, y.to(f8), y_scale=torch.zeros(4, 3))
    x8, w8 = torch.zeros(4, 256).to(f8), torch.zeros(100, 256).to(f8)
    xs, ws, o = torch.zeros(4, 2), torch.zeros(1, 2), torch.zeros(4, 100)
    refused(vxb.fp8_product, x8, xs, w8, ws, o)
    refused(vxb.fp8_product, x, xs, w8, ws, o)
    refused(vxb.fp8_product, x8, xs[:, :1], w8, ws, o)
    refused(vxb.fp8_product, x8, xs, w8, torch.zeros(2, 2), o)
    refused(vxb.fp8_product, x8, xs, w8, ws, o, bias=torch.zeros(99))
    q, k, pos, f = torch.zeros(4, 4, 64), torch.zeros(4, 2, 64), torch.zeros(4, dtype=torch.int64), torch.zeros(32)
    refused(vxb.rotary, q, pos, f, q, k=k, k_out=k)
    refused(vxb.rotary, q, pos.int(), f, q)
    refused(vxb.rotary, q, pos, f.double(), q)
    refused(vxb.rotary, q, pos, f, q, k=k)
    c = torch.zeros(3, 16, 2, 64)
    refused(vxb.rotary_append, q, k, k, pos, pos, f, q, c, c)
    refused(vxb.rotary_append, q, k, k, pos, pos.int(), f, q, c, c)
    refused(vxb.rotary_append, q, k, k, pos, pos, f, q, c, c.transpose(0, 1).contiguous().transpose(0, 1))
    i = torch.zeros(3, dtype=torch.int32)
    h, ch, t = q.half(), c.half(), torch.zeros(2, 1, dtype=torch.int32)
    refused(vxb.paged_attention, h, ch, ch, t, i, i[:2], h)
    refused(vxb.paged_attention, h, ch, ch, t.long(), i, i[:2], h)
    refused(vxb.paged_attention, h, ch, ch, t, i[:2], i[:2], h)
    refused(vxb.paged_attention, h, c, c, t, i, i[:2], h)


def test_rotary_frequencies():
    f, factor = vxb.rotary_frequencies(8, base=100.0)
    assert f.dtype.name == "float32" and factor == 1.0
    assert [float(v) for v in f] == pytest.approx([1.0, 100.0 ** -0.25, 0.1, 100.0 ** -0.75], rel=2 ** -23)
    g, factor = vxb.rotary_frequencies(8, base=100.0, linear=4.0)
    assert list(g) == pytest.approx([float(v) / 4 for v in f], rel=2 ** -23) and factor == 1.0
    g, factor = vxb.rotary_frequencies(8, base=100.0, factors=[1, 2, 4, 8], original_length=4096, length=4096 ** 2)
    assert list(g) == pytest.approx([float(v) / d for v, d in zip(f, (1, 2, 4, 8))], rel=2 ** -23)
    assert factor == pytest.approx(2 ** 0.5)  # ln(length / original) = ln(original)
    assert vxb.rotary_frequencies(8, factors=[1] * 4, original_length=4096, length=4096)[1] == 1.0
    for bad in (dict(R=7), dict(R=0), dict(R=8, factors=[1, 2])):
        with pytest.raises(ValueError):
            vxb.rotary_frequencies(**bad)


def test_entry_arguments_match_their_signatures():
    for name, a in (("rms_norm", NORM), ("fp8_product", PROD), ("rotary", ROT), ("rotary_append", APPEND),
                    ("paged_attention", ATTN)):
        assert len(a) == len(vxb.SIGNATURES["vxb_" + name][1])
    assert ctypes.sizeof(ctypes.c_void_p) == 8


def test_operators_sync_refuses():
    assert vxb.lib().vxb_operators_sync(-1, None) == vxb.ERR_INVALID_ARGUMENT
    for bad in (0, -3, 2000001):
        assert vxb.lib().vxb_debug_operators_wait_probe(bad, None) == vxb.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("name,base,change", [
    ("rotary", "ROT", dict(qot=0)), ("rotary", "ROT", dict(qoh=0)), ("rotary", "ROT", dict(qoh=32)),
    ("rotary", "ROT", dict(qot=192)), ("rotary", "ROT", dict(kot=64)), ("rotary", "ROT", dict(koh=-63)),
    ("rotary_append", "APPEND", dict(qoh=0)), ("rotary_append", "APPEND", dict(ps=0)),
    ("rotary_append", "APPEND", dict(ss=64)), ("rotary_append", "APPEND", dict(hs=32)),
    ("rotary_append", "APPEND", dict(ps=1024)), ("paged_attention", "ATTN", dict(ot=0)),
    ("paged_attention", "ATTN", dict(oh=0)), ("paged_attention", "ATTN", dict(oh=56)),
    ("paged_attention", "ATTN", dict(ot=64)), ("paged_attention", "ATTN", dict(ot=2 ** 62, oh=1))])
def test_outputs_whose_heads_overlap_are_refused(name, base, change):
    """(Threads would race for one place.)"""
    assert rc(name, *{**globals()[base], **change}.values()) == vxb.ERR_INVALID_ARGUMENT
    assert b"overlap" in vxb.lib().vxb_last_error()


@pytest.mark.parametrize("scale", [2.4e38, -3e38])
def test_attention_scale_that_overflows_in_log2_units_is_refused(scale):
    """(Scores of 0 would become 0 * inf.)"""
    assert rc("paged_attention", *{**ATTN, "scale": scale}.values()) == vxb.ERR_INVALID_ARGUMENT


def test_wrappers_refuse_lazily_negated_views():
    """Their memory holds the values with the other sign."""
    x, w, y = torch.zeros(4, 256), torch.zeros(256), torch.zeros(4, 256)
    for a in ((torch._neg_view(x), w, y), (x, torch._neg_view(w), y), (x, w, torch._neg_view(y))):
        with pytest.raises(vxb.VxbError, match="negated"):
            vxb.rms_norm(*a)
