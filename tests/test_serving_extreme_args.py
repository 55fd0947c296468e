"""Refusals of the operators over several sequences beside those of test_serving_args.py.  CPU only."""
import pytest

from heliopause_amd import hip_kernels as H
from test_serving_args import ARG, INF, NAN, attention, cache, rules


def test_reserved_field():
    assert H.lib().hp_hip_paged_attention_device(cache(), attention(reserved=1), None) == ARG
    assert "reserved" in H.last_error()


@pytest.mark.parametrize("cap", [-1.0, NAN, INF, -INF])
def test_softcaps_of_the_rules(cap):
    assert H.lib().hp_hip_logit_rules_device(rules(softcap=cap), None) == ARG
    assert "softcap" in H.last_error()
