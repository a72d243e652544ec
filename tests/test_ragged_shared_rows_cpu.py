"""The ragged-batch entries refuse outputs and caches whose rows are one memory (strides of 0, as of
an expanded tensor): sequences, heads or tokens would write over one another."""
import pytest

from halftone_quantizedkvcache_b200 import _lib
from test_ragged_cpu import (CODES, D, HKV, HQ, INVALID, S, WORKSPACE, decode_args, prefill_args, prefix_args,
                             rope_args)


@pytest.mark.parametrize("change,code", [
    (dict(os=(0, D, 1)), INVALID), (dict(os=(HQ * D, 0, 1)), INVALID),
    (dict(os=(0, D, 1), B=1), WORKSPACE),              # one sequence: its stride is never used
    (dict(qs=(0, D, 1), kvs=(0, S * D, D)), WORKSPACE),  # what is only read may be shared
])
def test_window_decode(change, code):
    assert _lib.lib().hq_window_decode_int8(*decode_args(**change)) == code


@pytest.mark.parametrize("change,code", [
    (dict(os=(0, D, HQ * D, 1)), INVALID), (dict(os=(HQ * 40 * D, 0, HQ * D, 1)), INVALID),
    (dict(os=(HQ * 40 * D, D, 0, 1)), INVALID), (dict(qs=(0, 40 * D, D, 1)), WORKSPACE),
])
def test_window_prefill(change, code):
    assert _lib.lib().hq_window_prefill_int8(*prefill_args(**change)) == code


@pytest.mark.parametrize("change,code", [
    (dict(os=(0, D, 1)), INVALID), (dict(os=(HQ * D, 0, 1)), INVALID),
    (dict(qs=(0, D, 1), pkvs=(0, S * D, D)), WORKSPACE),
])
def test_prefix_decode(change, code):
    assert _lib.lib().hq_prefix_decode_int8(*prefix_args(**change)) == code


@pytest.mark.parametrize("change", [
    dict(qos=(0, 3 * D, D, 1)), dict(qos=(HQ * 3 * D, 0, D, 1)), dict(qos=(HQ * 3 * D, 3 * D, 0, 1)),
    dict(cs=(0, S * D, D)), dict(cs=(HKV * S * D, 0, D)), dict(cs=(HKV * S * D, S * D, 0)),
    dict(vss=(0, S, 1)), dict(vss=(HKV * S, 0, 1)), dict(vss=(HKV * S, S, 0)),
])
def test_rope_append(change):
    assert _lib.lib().hq_rope_append_kv(*rope_args(**change)) == INVALID


def test_rope_append_takes_the_strides_of_single_extents():
    one = dict(B=1, Hq=1, Hkv=1, S=0, cap=1, qos=(0, 0, 0, 1), cs=(0, 0, 0), vss=(0, 0, 0))
    assert _lib.lib().hq_rope_append_kv(*rope_args(**one)) == _lib.OK
