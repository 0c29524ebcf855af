"""Argument errors of the mixture-of-experts operators are reported before any device call (no GPU), and calls with
nothing to do succeed."""
import ctypes as C

import pytest

from helpers import pkg

FAKE = 1 << 20  # never dereferenced: every check fails before a device call


def error(name, *args):
    L = pkg().lib()
    getattr(L, name)(*args)
    return L.tinymlp_last_error_message().decode() if L.tinymlp_last_error() else ""


def route_option(**kw):
    o = dict(numExperts=8, topK=2, scoreType=0, numGroups=1, topGroups=1, groupScore=2, renormalize=1, scale=1.0, logitsType=0)
    o.update(kw)
    return pkg().RouteOption(**o)


@pytest.mark.parametrize("change,text", [
    (dict(numExperts=0), "numExperts"), (dict(numExperts=1025), "numExperts"), (dict(topK=0), "topK"), (dict(topK=9), "topK"),
    (dict(numExperts=64, topK=33), "topK"), (dict(scoreType=2), "scoreType"), (dict(numGroups=3), "numGroups"),
    (dict(numGroups=0), "numGroups"), (dict(numExperts=130, numGroups=65), "numGroups"), (dict(numGroups=4, topGroups=5), "topGroups"),
    (dict(numGroups=4, topGroups=0), "topGroups"), (dict(numGroups=4, topGroups=2, groupScore=3), "groupScore"),
    (dict(scale=float("nan")), "scale"), (dict(logitsType=3), "type")])
def test_route_options(change, text):
    o = route_option(**change)
    assert text in error("launchRouteExperts", C.byref(o), FAKE, 2000, None, FAKE, FAKE, 4, None)
    assert text in error("launchRouteExpertsBackward", C.byref(o), FAKE, 2000, FAKE, FAKE, FAKE, 2000, 4, None)


def test_route_arguments():
    o = C.byref(route_option())
    assert "null" in error("launchRouteExperts", None, FAKE, 8, None, FAKE, FAKE, 4, None)
    assert "null" in error("launchRouteExperts", o, None, 8, None, FAKE, FAKE, 4, None)
    assert "null" in error("launchRouteExperts", o, FAKE, 8, None, None, FAKE, 4, None)
    assert "null" in error("launchRouteExperts", o, FAKE, 8, None, FAKE, None, 4, None)
    assert "Stride" in error("launchRouteExperts", o, FAKE, 7, None, FAKE, FAKE, 4, None)
    assert "numTokens" in error("launchRouteExperts", o, FAKE, 8, None, FAKE, FAKE, -1, None)
    assert "numTokens" in error("launchRouteExperts", o, FAKE, 8, None, FAKE, FAKE, (1 << 30) + 1, None)
    assert error("launchRouteExperts", o, None, 8, None, None, None, 0, None) == ""
    assert "null" in error("launchRouteExpertsBackward", o, FAKE, 8, FAKE, None, FAKE, 8, 4, None)
    assert "null" in error("launchRouteExpertsBackward", o, FAKE, 8, FAKE, FAKE, None, 8, 4, None)
    assert "Stride" in error("launchRouteExpertsBackward", o, FAKE, 8, FAKE, FAKE, FAKE, 7, 4, None)
    assert error("launchRouteExpertsBackward", o, None, 8, None, None, None, 8, 0, None) == ""


def test_plan():
    L = pkg().lib()
    cap = L.routePlanCapacity
    assert cap(0, 1, 8, 128) == 0 and cap(1, 1, 8, 128) == 128 and cap(100, 2, 8, 1) == 200
    assert cap(100, 2, 8, 128) == -(-(200 + 8 * 127) // 128) * 128
    for bad in ((-1, 1, 8, 1), (1, 0, 8, 1), (1, 33, 8, 1), (1, 1, 0, 1), (1, 1, 1025, 1), (1, 1, 8, 0), (1, 1, 8, 129),
                (1 << 29, 4, 8, 1)):
        assert cap(*bad) == -1
        assert "numTokens" in error("launchRoutePlan", FAKE, *bad, 1 << 30, FAKE, FAKE, FAKE, None)
    assert "capacity" in error("launchRoutePlan", FAKE, 100, 2, 8, 128, cap(100, 2, 8, 128) - 1, FAKE, FAKE, FAKE, None)
    for hole in (0, 6, 7, 8):
        args = [FAKE, 100, 2, 8, 1, 200, FAKE, FAKE, FAKE, None]
        args[hole] = None
        assert "null" in error("launchRoutePlan", *args)


def quant_option(**kw):
    o = dict(rows=4, cols=100, batch=1, blockRows=1, srcType=0, slotsPerRow=1, srcRows=4, srcStride=100, srcBatchStride=0,
             gateStride=100)
    o.update(kw)
    return pkg().Fp8QuantOption(**o)


@pytest.mark.parametrize("change,args,text", [
    (dict(rows=-1), {}, "rows"), (dict(cols=0), {}, "cols"), (dict(cols=(1 << 22) + 1), {}, "cols"), (dict(batch=0), {}, "batch"),
    (dict(blockRows=64), {}, "blockRows"), (dict(srcType=9), {}, "type"), (dict(srcStride=99), {}, "srcStride"),
    (dict(gateStride=99), dict(gate=FAKE), "gateStride"), (dict(slotsPerRow=0), dict(order=FAKE), "slotsPerRow"),
    (dict(batch=2), dict(order=FAKE), "order"), ({}, dict(weights=FAKE), "weights"), (dict(batch=2), dict(gate=FAKE), "gate"),
    (dict(srcRows=3), {}, "srcRows"), ({}, dict(q=None, s=None), "q or qt"), ({}, dict(s=None), "scales"),
    ({}, dict(qt=FAKE), "scales"), ({}, dict(q=FAKE + 8), "aligned"), ({}, dict(src=None), "null"),
    (dict(batch=2, srcBatchStride=-1), {}, "srcBatchStride")])
def test_quantize(change, args, text):
    a = dict(src=FAKE, order=None, weights=None, gate=None, q=FAKE, s=FAKE, qt=None, st=None)
    a.update(args)
    assert text in error("launchFp8Quantize", C.byref(quant_option(**change)), *a.values(), None)
    assert "null" in error("launchFp8Quantize", None, *a.values(), None)


def test_nothing_to_quantize_or_multiply():
    assert error("launchFp8Quantize", C.byref(quant_option(rows=0)), None, None, None, None, FAKE, FAKE, None, None, None) == ""
    assert error("launchFp8Product", C.byref(product_option(m=0)), None, None, None, None, None, None, None) == ""


def product_option(**kw):
    o = dict(m=4, n=8, k=100, numExperts=1, grouping=0, scaleRowsB=128, activation=0, outType=0, outStride=8)
    o.update(kw)
    return pkg().Fp8ProductOption(**o)


@pytest.mark.parametrize("change,args,text", [
    (dict(m=-1), {}, "m must"), (dict(n=0), {}, "n must"), (dict(k=0), {}, "k 1"), (dict(k=(1 << 22) + 1), {}, "k 1"),
    (dict(grouping=3), {}, "grouping"), (dict(numExperts=2), {}, "numExperts"), (dict(numExperts=0), {}, "numExperts"),
    (dict(grouping=1, numExperts=1025), dict(offsets=FAKE), "numExperts"), (dict(scaleRowsB=2), {}, "scaleRowsB"),
    (dict(activation=2), {}, "activation"), (dict(outType=-1), {}, "type"), (dict(outStride=7), {}, "outStride"),
    ({}, dict(offsets=FAKE), "offsets"), (dict(grouping=1), {}, "offsets"), (dict(grouping=2), {}, "offsets"),
    ({}, dict(a=None), "null"), ({}, dict(a_s=None), "null"), ({}, dict(b=None), "null"), ({}, dict(b_s=None), "null"),
    ({}, dict(out=None), "null"), ({}, dict(a=FAKE + 4), "aligned"), ({}, dict(b=FAKE + 8), "aligned"),
    ({}, dict(a_s=FAKE + 1), "aligned"), ({}, dict(b_s=FAKE + 2), "aligned")])
def test_product(change, args, text):
    a = dict(a=FAKE, a_s=FAKE, b=FAKE, b_s=FAKE, offsets=None, out=FAKE)
    a.update(args)
    assert text in error("launchFp8Product", C.byref(product_option(**change)), *a.values(), None)
    assert "null" in error("launchFp8Product", None, *a.values(), None)


def test_combine():
    def fwd(dim=8, type_=0, rows=FAKE, n=4, rs=8, pos=FAKE, w=None, out=FAKE, os_=8, T=4, k=2):
        return error("launchExpertCombine", dim, type_, rows, n, rs, pos, w, out, os_, T, k, None)

    def bwd(dim=8, type_=0, rows=FAKE, n=4, rs=8, pos=FAKE, dout=FAKE, os_=8, dw=FAKE, T=4, k=2):
        return error("launchExpertCombineBackward", dim, type_, rows, n, rs, pos, dout, os_, dw, T, k, None)

    for f in (fwd, bwd):
        assert "dim" in f(dim=0) and "type" in f(type_=5) and "numRows" in f(n=-1) and "topK" in f(k=0) and "topK" in f(k=33)
        assert "strides" in f(rs=7) and "strides" in f(os_=7) and "null" in f(rows=None) and "null" in f(pos=None)
        assert "numTokens" in f(T=-1) and f(T=0, rows=None, pos=None) == ""
    assert "null" in fwd(out=None) and "null" in bwd(dout=None) and "null" in bwd(dw=None)


def norm_option(**kw):
    o = dict(dim=8, postNorm=1, preNorm=1, gateRows=0, residualScale=1.0, blockScale=1.0, epsilon=1e-6, dataType=0, strideX=8,
             strideF=8, strideGate=8, strideY=8, strideH=8)
    o.update(kw)
    return pkg().NormGateOption(**o)


@pytest.mark.parametrize("change,args,text", [
    (dict(dim=0), {}, "dim"), (dict(dim=8193), {}, "dim"), (dict(postNorm=3), {}, "norm"), (dict(preNorm=-1), {}, "norm"),
    (dict(dataType=3), {}, "type"), (dict(gateRows=-1), {}, "gateRows"), (dict(epsilon=-1.0), {}, "epsilon"),
    ({}, dict(f=None), "need f"), (dict(gateRows=1, postNorm=0), dict(f=None), "need f"), (dict(gateRows=2), {}, "gate"),
    ({}, dict(gate=FAKE), "gate"), (dict(postNorm=0), dict(pw=FAKE), "post"), (dict(preNorm=0), dict(nb=FAKE), "pre"),
    (dict(strideX=7), {}, "strides"), (dict(strideF=7), {}, "strides"), (dict(gateRows=1, strideGate=7), dict(gate=FAKE), "strides"),
    (dict(strideY=7), {}, "strides"), (dict(strideH=7), {}, "strides"), ({}, dict(x=None), "null")])
def test_norm(change, args, text):
    a = dict(x=FAKE, f=FAKE, gate=None, pw=None, pb=None, nw=None, nb=None)
    a.update(args)
    o = C.byref(norm_option(**change))
    assert text in error("launchNormGateResidual", o, *a.values(), FAKE, FAKE, 4, None)
    assert text in error("launchNormGateResidualBackward", o, *a.values(), FAKE, FAKE, *[None] * 7, 4, None)


def test_norm_outputs():
    a = [FAKE, FAKE] + [None] * 5
    o = C.byref(norm_option())
    assert "NULL" in error("launchNormGateResidual", o, *a, None, None, 4, None)
    assert "numRows" in error("launchNormGateResidual", o, *a, FAKE, FAKE, -1, None)
    assert error("launchNormGateResidual", o, *a, FAKE, FAKE, 0, None) == ""
    assert "null" in error("launchNormGateResidual", None, *a, FAKE, FAKE, 4, None)
    assert "gate" in error("launchNormGateResidualBackward", o, *a, FAKE, FAKE, None, None, FAKE, None, None, None, None, 4, None)
    o = C.byref(norm_option(postNorm=0, preNorm=0))
    assert "post norm" in error("launchNormGateResidualBackward", o, *a, FAKE, FAKE, None, None, None, FAKE, None, None, None, 4, None)
    assert "pre norm" in error("launchNormGateResidualBackward", o, *a, FAKE, FAKE, None, None, None, None, None, None, FAKE, 4, None)
    b = [FAKE, None] + [None] * 5
    assert "need f" in error("launchNormGateResidualBackward", o, *b, FAKE, FAKE, None, FAKE, None, None, None, None, None, 4, None)
