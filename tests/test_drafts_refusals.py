"""Refusals of the drafted-token operators: arguments are checked before the device is
needed, so these run without a GPU."""
import ctypes

import pytest

import g4hip

INF = float("inf")
NAN = float("nan")


def refused(rc, *words):
    assert rc == g4hip.G4_E_ARG
    msg = g4hip.lib().g4_last_error().decode()
    for w in words:
        assert w in msg, msg


@pytest.mark.parametrize("nodes,heads,hd,prefix,sliding,window", [
    (-1, 8, 256, 0, 0, 0), (257, 8, 256, 0, 0, 0), (4, 0, 256, 0, 0, 0), (4, 9, 256, 0, 0, 0),
    (4, 8, 96, 0, 0, 0), (4, 8, 1024, 0, 0, 0), (4, 8, 0, 0, 0, 0), (4, 8, 256, -1, 0, 0),
    (4, 8, 256, 0x7fffffff, 0, 0), (4, 8, 256, 10, 1, 0), (4, 8, 256, 10, 1, -5)])
def test_attention_tree(nodes, heads, hd, prefix, sliding, window):
    refused(g4hip.lib().g4_attention_tree(8, 8, 8, nodes, heads, hd, prefix, 8, sliding, window, 8),
            "g4_attention_tree")


@pytest.mark.parametrize("n,E,rows,k,stride", [
    (-1, 16, 8, 64, 8), (2, 16, -1, 64, 8), (2, 16, 8, 0, 8), (2, 16, 8, 12, 8), (2, 16, 8, 4104, 8),
    (2, 16, 8, 64, 7), (2, 8, 8, 64, 8), (65537, 16, 8, 64, 8),
    (2, 16, (1 << 30) + 1, 64, 1 << 31), (3, 16, 8, 64, 1 << 61), (2, 16, 8, 64, (1 << 64) - 1)])
def test_head_rows(n, E, rows, k, stride):
    refused(g4hip.lib().g4_bf16_head_rows(16, n, E, rows, k, 16, stride, 1.0, 30.0),
            "g4_bf16_head_rows")


@pytest.mark.parametrize("rows,vocab,stride,t,k,p,m", [
    (-1, 10, 10, 1, 0, 1, 0), (1, 0, 10, 1, 0, 1, 0), (1, 10, 9, 1, 0, 1, 0),
    (1, 10, 10, -0.5, 0, 1, 0), (1, 10, 10, INF, 0, 1, 0), (1, 10, 10, NAN, 0, 1, 0),
    (1, 10, 10, 1, -1, 1, 0), (1, 10, 10, 1, 0, 0, 0), (1, 10, 10, 1, 0, 1.5, 0),
    (1, (1 << 22) + 1, 1 << 25, 1, 0, 1, 0), (1, 10, 10, 1, 0, NAN, 0), (1, 10, 10, 1, 0, 1, -0.1), (1, 10, 10, 1, 0, 1, 1.1),
    (1, 10, 10, 1, 0, 1, NAN), (3, 10, 1 << 61, 1, 0, 1, 0), (2, 10, (1 << 64) - 1, 1, 0, 1, 0)])
def test_sample(rows, vocab, stride, t, k, p, m):
    params = g4hip.SampleParams(t, k, p, m)
    refused(g4hip.lib().g4_sample(8, stride, rows, vocab, ctypes.byref(params), 8, 8, None),
            "g4_sample")


def test_sample_without_params():
    refused(g4hip.lib().g4_sample(8, 8, 1, 8, None, 8, 8, None), "params")


@pytest.mark.parametrize("planes,width,n,dst_row,src_rows", [
    (0, 8, 1, 0, 4), (129, 8, 1, 0, 4), (1, 0, 1, 0, 4), (1, (1 << 24) + 1, 1, 0, 4),
    (2, 0x7fffffff, 0x7fffffff, 0x7fffffff, 0x7fffffff), (1, -8, 1, 0, 4), (1, 8, -1, 0, 4),
    (1, 8, 1, -1, 4), (1, 8, 1, 0, -1), (1, 8, 1, 0, 0)])
def test_cache_rows(planes, width, n, dst_row, src_rows):
    p = (ctypes.c_void_p * 129)(*[16] * 129)
    w = (ctypes.c_int * 129)(*[width] * 129)
    refused(g4hip.lib().g4_cache_rows(p, p, w, planes, 8, n, dst_row, src_rows), "g4_cache_rows")


def test_cache_rows_null_arrays():
    p = (ctypes.c_void_p * 1)(16)
    w = (ctypes.c_int * 1)(8)
    for a in ((None, p, w), (p, None, w), (p, p, None)):
        refused(g4hip.lib().g4_cache_rows(*a, 1, 8, 1, 0, 4), "null")


def test_cache_planes_of_different_counts():
    with pytest.raises(ValueError):
        g4hip.CachePlanes([8, 8], [8], [4])
