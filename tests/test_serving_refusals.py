"""Argument errors of the 4-bit products, the expert layer and the gradients' norm are reported before any device call (no
GPU), and calls with nothing to do succeed."""
import ctypes as C
import math

import pytest

from helpers import pkg

FAKE = 1 << 20  # never dereferenced: every check fails before a device call


def error(name, *args):
    L = pkg().lib()
    getattr(L, name)(*args)
    return L.tinymlp_last_error_message().decode() if L.tinymlp_last_error() else ""


def test_pitches():
    P = pkg()
    assert [P.fp4_pitch(c) for c in (1, 128, 129, 4096)] == [64, 64, 128, 2048]
    assert [P.fp4_scale_pitch(c) for c in (1, 128, 129, 4096)] == [4, 4, 8, 128]


def quant_option(**kw):
    o = dict(rows=4, cols=100, batch=1, scaleRule=0, srcType=0, slotsPerRow=1, srcRows=4, srcStride=100, srcBatchStride=0)
    o.update(kw)
    return pkg().Fp4QuantOption(**o)


@pytest.mark.parametrize("change,args,text", [
    (dict(rows=-1), {}, "rows"), (dict(rows=(1 << 30) + 1), {}, "rows"), (dict(cols=0), {}, "cols"),
    (dict(cols=(1 << 22) + 1), {}, "cols"), (dict(batch=0), {}, "batch"), (dict(batch=65536), {}, "batch"),
    (dict(scaleRule=2), {}, "scaleRule"), (dict(srcType=9), {}, "type"), (dict(srcStride=99), {}, "srcStride"),
    (dict(slotsPerRow=0), dict(order=FAKE), "slotsPerRow"), (dict(batch=2), dict(order=FAKE), "order"),
    (dict(srcRows=3), {}, "srcRows"), (dict(srcRows=-1), {}, "srcRows"), (dict(batch=2, srcBatchStride=-1), {}, "srcBatchStride"),
    ({}, dict(q=None), "null"), ({}, dict(s=None), "null"), ({}, dict(src=None), "null"), ({}, dict(q=FAKE + 8), "aligned"),
    ({}, dict(s=FAKE + 2), "aligned")])
def test_quantize(change, args, text):
    a = dict(src=FAKE, order=None, q=FAKE, s=FAKE)
    a.update(args)
    assert text in error("launchFp4Quantize", C.byref(quant_option(**change)), *a.values(), None)
    assert "null" in error("launchFp4Quantize", None, *a.values(), None)


def product_option(**kw):
    o = dict(m=4, n=8, k=100, numExperts=1, grouping=0, activation=0, outType=0, outStride=8)
    o.update(kw)
    return pkg().Fp4ProductOption(**o)


@pytest.mark.parametrize("change,args,text", [
    (dict(m=-1), {}, "m must"), (dict(n=0), {}, "n and k"), (dict(k=0), {}, "n and k"), (dict(k=(1 << 22) + 1), {}, "n and k"),
    (dict(grouping=2), dict(offsets=FAKE), "grouping"), (dict(grouping=-1), {}, "grouping"), (dict(numExperts=2), {}, "numExperts"),
    (dict(numExperts=0), {}, "numExperts"), (dict(grouping=1, numExperts=1025), dict(offsets=FAKE), "numExperts"),
    (dict(activation=2), {}, "activation"), (dict(outType=0x100), {}, "type"), (dict(outStride=7), {}, "outStride"),
    ({}, dict(offsets=FAKE), "offsets"), (dict(grouping=1), {}, "offsets"), ({}, dict(a=None), "null"),
    ({}, dict(a_s=None), "null"), ({}, dict(b=None), "null"), ({}, dict(b_s=None), "null"), ({}, dict(out=None), "null"),
    ({}, dict(a=FAKE + 4), "aligned"), ({}, dict(b=FAKE + 8), "aligned"), ({}, dict(a_s=FAKE + 1), "aligned"),
    ({}, dict(b_s=FAKE + 2), "aligned")])
def test_product(change, args, text):
    a = dict(a=FAKE, a_s=FAKE, b=FAKE, b_s=FAKE, offsets=None, out=FAKE)
    a.update(args)
    assert text in error("launchFp4Product", C.byref(product_option(**change)), *a.values(), None)
    assert "null" in error("launchFp4Product", None, *a.values(), None)


def layer_option(route=None, **kw):
    P = pkg()
    r = dict(numExperts=8, topK=2, scoreType=0, numGroups=1, topGroups=1, groupScore=2, renormalize=1, scale=1.0, logitsType=0)
    r.update(route or {})
    o = dict(dim=64, hidden=96, activation=1, gated=0, weightFormat=0, scaleRows=128, dataType=2, routerType=0, strideX=64,
             strideOut=64)
    o.update(kw)
    return P.ExpertLayerOption(route=P.RouteOption(**r), **o)


@pytest.mark.parametrize("route,change,args,text", [
    (dict(numExperts=0), {}, {}, "numExperts"), (dict(numExperts=1025), {}, {}, "numExperts"), (dict(topK=0), {}, {}, "topK"),
    (dict(topK=9), {}, {}, "topK"), (dict(scoreType=2), {}, {}, "scoreType"), (dict(numGroups=3), {}, {}, "numGroups"),
    (dict(numGroups=4, topGroups=5), {}, {}, "topGroups"), (dict(scale=math.inf), {}, {}, "scale"),
    (dict(logitsType=1), {}, {}, "logitsType"), ({}, dict(dim=0), {}, "dim"), ({}, dict(dim=16385), {}, "dim"),
    ({}, dict(hidden=0), {}, "hidden"), ({}, dict(hidden=16385), {}, "hidden"), ({}, dict(activation=4), {}, "activation"),
    ({}, dict(activation=-1), {}, "activation"), ({}, dict(weightFormat=2), {}, "weightFormat"),
    ({}, dict(scaleRows=64), {}, "scaleRows"), ({}, dict(weightFormat=1), {}, "scaleRows"), ({}, dict(dataType=3), {}, "type"),
    ({}, dict(routerType=-1), {}, "type"), ({}, dict(strideX=63), {}, "strides"), ({}, dict(strideOut=63), {}, "strides"),
    ({}, {}, dict(tokens=65), "numTokens"), ({}, {}, dict(tokens=-1), "numTokens"), ({}, {}, dict(x=None), "null"),
    ({}, {}, dict(router=None), "null"), ({}, {}, dict(w1=None), "null"), ({}, {}, dict(s1=None), "null"),
    ({}, {}, dict(w2=None), "null"), ({}, {}, dict(s2=None), "null"), ({}, {}, dict(out=None), "null"),
    ({}, {}, dict(w1=FAKE + 8), "aligned"), ({}, {}, dict(w2=FAKE + 4), "aligned"), ({}, {}, dict(s1=FAKE + 2), "aligned"),
    ({}, {}, dict(s2=FAKE + 1), "aligned")])
def test_layer(route, change, args, text):
    a = dict(x=FAKE, router=FAKE, bias=None, w1=FAKE, s1=FAKE, w2=FAKE, s2=FAKE, out=FAKE + (1 << 20), tokens=4)
    a.update(args)
    assert text in error("launchExpertLayer", C.byref(layer_option(route, **change)), *a.values(), None)
    assert "null" in error("launchExpertLayer", None, *a.values(), None)


def test_nothing_to_do():
    assert error("launchFp4Quantize", C.byref(quant_option(rows=0)), None, None, None, None, None) == ""
    assert error("launchFp4Product", C.byref(product_option(m=0)), None, None, None, None, None, None, None) == ""
    assert error("launchExpertLayer", C.byref(layer_option()), *[None] * 8, 0, None) == ""


def tensors(*items):
    P = pkg()
    return (P.GradTensor * len(items))(*(P.GradTensor(data=d, out=o, n=n, dataType=t) for d, o, n, t in items))


@pytest.mark.parametrize("item,text", [
    ((FAKE, None, -1, 0), "n must"), ((FAKE, None, (1 << 40) + 1, 0), "n must"), ((None, None, 4, 0), "null"),
    ((FAKE, None, 4, 3), "type"), ((FAKE + 2, None, 4, 0), "aligned"), ((FAKE + 1, None, 4, 1), "aligned"),
    ((FAKE, FAKE + (1 << 16) + 2, 4, 0), "aligned")])
def test_lists(item, text):
    t = tensors((FAKE + (1 << 18), None, 8, 0), item)
    assert text in error("launchGradNorm", t, 2, 0, 1.0, FAKE, None)
    assert text in error("launchGradClip", t, 2, 1.0, 0, FAKE, None)
    assert text in error("launchGradNormClip", t, 2, 0, 1.0, 1.0, 0, FAKE, None)


def test_gradients():
    t = tensors((FAKE, None, 8, 0))
    for count, text in ((-1, "count"), (65537, "count")):
        assert text in error("launchGradNorm", t, count, 0, 1.0, FAKE, None)
        assert text in error("launchGradClip", t, count, 1.0, 0, FAKE, None)
    assert "null" in error("launchGradNorm", None, 1, 0, 1.0, FAKE, None)
    assert "null" in error("launchGradNorm", t, 1, 0, 1.0, None, None)
    assert "null" in error("launchGradClip", t, 1, 1.0, 0, None, None)
    assert "null" in error("launchGradNormClip", t, 1, 0, 1.0, 1.0, 0, None, None)
    for scale in (0.0, -1.0, math.inf, math.nan):
        assert "gradScale" in error("launchGradNorm", t, 1, 0, scale, FAKE, None)
        assert "gradScale" in error("launchGradNormClip", t, 1, 0, scale, 1.0, 0, FAKE, None)
    for m in (-1.0, math.nan):
        assert "maxNorm" in error("launchGradClip", t, 1, m, 0, FAKE, None)
        assert "maxNorm" in error("launchGradNormClip", t, 1, 0, 1.0, m, 0, FAKE, None)
    assert "norm" in error("launchGradNorm", t, 1, 2, 1.0, FAKE, None)
    assert "nonFinite" in error("launchGradClip", t, 1, 1.0, 2, FAKE, None)
    assert error("launchGradClip", None, 0, 1.0, 0, FAKE, None) == ""


@pytest.mark.parametrize("items", [
    [(FAKE, None, 8, 0), (FAKE, None, 8, 0)], [(FAKE, None, 8, 0), (FAKE + 28, None, 8, 0)],
    [(FAKE + 16, None, 8, 1), (FAKE, None, 8, 0)], [(FAKE, FAKE + 4, 8, 0)], [(FAKE, FAKE + 64, 8, 0), (FAKE + 68, None, 8, 0)],
    [(FAKE, FAKE + 64, 8, 0), (FAKE + 32, FAKE + 64, 8, 0)], [(FAKE, None, 100, 0), (FAKE + 8, FAKE + 4096, 4, 0)]])
def test_what_is_written_overlaps_nothing(items):
    for order in (items, items[::-1]):
        t = tensors(*order)
        assert "overlaps" in error("launchGradClip", t, len(order), 1.0, 0, FAKE, None)
        assert "overlaps" in error("launchGradNormClip", t, len(order), 0, 1.0, 1.0, 0, FAKE, None)
