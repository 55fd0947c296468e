"""Refusals of the operators over several sequences beside those of test_serving_args.py.  CPU only."""
from heliopause_amd import hip_kernels as H
from test_serving_args import ARG, attention, cache


def test_reserved_field():
    assert H.lib().hp_hip_paged_attention_device(cache(), attention(reserved=1), None) == ARG
    assert "reserved" in H.last_error()
