"""Tensors that lie over one another are refused by the operators for long and speculative answers where what one
workgroup writes would be what another reads; decided from the host's arguments, without a GPU."""
import ctypes as C
import os
import subprocess

import pytest

import curoaring as cr
from test_long_answers_abi import EVICT, INVALID, P, ROTARY, WEIGHTS, _cache, _filled

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_rows_over_rows():
    """csrc/rows.hpp against all pairs of rows of small tensors."""
    exe = os.path.join(ROOT, "tests", "cpp", "rows_check")
    assert os.path.exists(exe), "tests/cpp/rows_check is built by __graft_entry__.build()"
    r = subprocess.run([exe], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and "rows_check: OK" in r.stdout, r.stdout + r.stderr


@pytest.mark.parametrize("args", [
    dict(q_token_stride=512), dict(q_head_stride=128), dict(q_token_stride=64, q_head_stride=192),  # in place, other strides
    dict(q_out=P + 128), dict(q_out=P + 512), dict(q_out=P + 2),  # a head, a token, an element further
    dict(q=P + 1024), dict(q_out=P + 64, out_token_stride=512),
    dict(q_out=P + 65536, out_token_stride=64), dict(q_out=P + 65536, out_token_stride=128),  # over one another
    dict(q_out=P + 65536, out_token_stride=64, out_head_stride=128)])
def test_turned_queries_over_others(args):
    a = _filled(cr.PagedRotaryArgs, ROTARY, args)
    assert cr.load().cr_paged_rotary(C.byref(a), C.byref(_cache()), None) == INVALID
    assert b"lie over one another" in cr._lib.cr_last_error()


@pytest.mark.parametrize("args", [
    dict(weights_out_stride=68), dict(weights_stride=128), dict(d_weights_out=P + 16), dict(d_weights_out=P + 256),
    dict(d_weights=P + 252), dict(positions_out_stride=128), dict(d_positions_out=P + 4), dict(d_positions=P + 256),
    dict(weights_stride=128, weights_out_stride=128, d_weights_out=P + 252)])
def test_evicted_rows_over_others(args):
    a = _filled(cr.PagedEvictArgs, EVICT, args)
    assert cr.load().cr_paged_evict(C.byref(a), None) == INVALID
    assert b"lie over others" in cr._lib.cr_last_error()


@pytest.mark.parametrize("args", [dict(d_past=P, past_stride=68), dict(d_past=P, past_stride=64, out_stride=128),
                                  dict(d_past=P + 16, past_stride=64), dict(d_past=P + 256, past_stride=64),
                                  dict(d_past=P + 252, past_stride=128, out_stride=128)])
def test_weights_over_others(args):
    a = _filled(cr.PagedWeightsArgs, WEIGHTS, args)
    assert cr.load().cr_paged_weights(C.byref(a), C.byref(_cache()), None) == INVALID
    assert b"lie over others" in cr._lib.cr_last_error()
