"""Argument checks and index rules of the operators over several sequences.  CPU only: every call here is refused on
the host before a device is looked for."""
import shutil
import subprocess
from pathlib import Path

import pytest

from heliopause_amd import hip_kernels as H

ROOT = Path(__file__).resolve().parents[1]
P = 1 << 20  # a 16-byte aligned address that no call gets as far as reading


def test_index_rules(tmp_path):
    """hp_pages.h over bad page tables, odd batches and uneven shares (tests/paged_index.cpp)."""
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "paged_index"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "paged_index.cpp"), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def cache(**change):
    c = H.paged_cache(P, P, H.HP_ELEM_F16, page_count=4, page_size=16, head_count_kv=2, head_dim=64, d_pages=P,
                      d_lengths=P, sequence_count=3, pages_per_sequence=2)
    for name, value in change.items():
        setattr(c, name, value)
    return c


def append(**change):
    p = H.HipPagedAppend(d_q=P, d_k=P, d_v=P, d_q_out=P, token_count=3, head_count=4, out_type=H.HP_ELEM_F16,
                         rope_dims=64, rope_freq_base=1e4, epsilon=1e-6)
    for name, value in change.items():
        setattr(p, name, value)
    return p


def attention(**change):
    p = H.HipPagedAttention(d_q=P, d_output=P, head_count=4, q_type=H.HP_ELEM_F32, out_type=H.HP_ELEM_F32, scale=1.0)
    for name, value in change.items():
        setattr(p, name, value)
    return p


def packed(**change):
    p = H.HipPackedAttention(d_q=P, d_k=P, d_v=P, d_output=P, d_offsets=P, token_count=9, sequence_count=2,
                             head_count=4, head_count_kv=2, head_dim=64, type=H.HP_ELEM_F16, out_type=H.HP_ELEM_F16,
                             scale=1.0)
    for name, value in change.items():
        setattr(p, name, value)
    return p


def rules(**change):
    p = H.HipLogitRules(d_logits=P, d_output=P, rows=2, n=100)
    for name, value in change.items():
        setattr(p, name, value)
    return p


NAN, INF = float("nan"), float("inf")
SHAPE, HEADS, TYPE, ARG = H.HP_ERR_SHAPE, H.HP_ERR_HEADS, H.HP_ERR_TYPE, H.HP_ERR_ARG

BAD_CACHE = [({"type": 0}, TYPE), ({"type": 4}, TYPE), ({"type": -1}, TYPE), ({"head_dim": 96}, SHAPE),
             ({"head_dim": 0}, SHAPE), ({"head_count_kv": 0}, HEADS), ({"head_count_kv": -2}, HEADS),
             ({"page_size": 8}, SHAPE), ({"page_size": 24}, SHAPE), ({"page_size": 8192}, SHAPE),
             ({"page_size": -16}, SHAPE), ({"page_count": 0}, SHAPE), ({"sequence_count": -1}, SHAPE),
             ({"sequence_count": 65536}, SHAPE), ({"pages_per_sequence": 0}, SHAPE),
             ({"pages_per_sequence": (1 << 26) + 1}, SHAPE), ({"page_stride": 2047}, SHAPE),
             ({"page_stride": 2049}, ARG), ({"page_stride": 1 << 50}, SHAPE), ({"d_keys": None}, ARG),
             ({"d_values": None}, ARG), ({"d_pages": None}, ARG), ({"d_lengths": None}, ARG), ({"d_keys": P + 8}, ARG),
             ({"d_values": P + 2}, ARG), ({"type": 3, "key_scale": 0.0}, ARG), ({"type": 3, "value_scale": NAN}, ARG),
             ({"type": 3, "value_scale": -1.0}, ARG), ({"type": 3, "key_scale": INF}, ARG),
             ({"type": 3, "page_stride": 2056}, ARG)]


@pytest.mark.parametrize("change,code", BAD_CACHE)
def test_bad_caches(change, code):
    c = cache(**change)
    assert H.lib().hp_hip_paged_append_device(c, append(), None) == code
    assert H.lib().hp_hip_paged_attention_device(c, attention(), None) == code


@pytest.mark.parametrize("change,code", [
    ({"out_type": 3}, TYPE), ({"out_type": 9}, TYPE), ({"head_count": 3}, HEADS), ({"head_count": 0}, HEADS),
    ({"head_count": -2}, HEADS), ({"d_q": None}, ARG), ({"d_q_out": None}, ARG), ({"d_k": None}, ARG),
    ({"rope_dims": 12}, SHAPE), ({"rope_dims": 72}, SHAPE), ({"rope_dims": -8}, SHAPE), ({"rope_freq_base": 0.0}, ARG),
    ({"rope_freq_base": NAN}, ARG), ({"epsilon": -1.0}, ARG), ({"epsilon": INF}, ARG), ({"token_count": 2}, SHAPE),
    ({"token_count": (1 << 23) + 1, "d_offsets": P}, SHAPE), ({"q_stride": 255}, SHAPE), ({"q_stride": 258}, ARG),
    ({"k_stride": 127}, SHAPE), ({"v_stride": 130}, ARG), ({"v_stride": 1 << 48}, SHAPE), ({"d_q": P + 4}, ARG),
    ({"d_v": P + 8}, ARG), ({"d_k_out": P + 4}, ARG)])
def test_bad_appends(change, code):
    assert H.lib().hp_hip_paged_append_device(cache(), append(**change), None) == code


@pytest.mark.parametrize("change,code", [
    ({"head_count": 3}, HEADS), ({"head_count": 0}, HEADS), ({"head_count": 65536}, HEADS), ({"q_type": 3}, TYPE),
    ({"out_type": -1}, TYPE), ({"scale": 0.0}, ARG), ({"scale": -1.0}, ARG), ({"scale": NAN}, ARG),
    ({"sliding_window": -1}, ARG), ({"q_stride": 128}, SHAPE), ({"output_stride": 257}, ARG), ({"d_q": None}, ARG),
    ({"d_output": None}, ARG), ({"d_output": P + 4}, ARG)])
def test_bad_attentions(change, code):
    assert H.lib().hp_hip_paged_attention_device(cache(), attention(**change), None) == code


def test_more_steps_than_the_kernel_counts():
    c = cache(sequence_count=65535, pages_per_sequence=1 << 26, head_count_kv=4)
    assert H.lib().hp_hip_paged_attention_device(c, attention(), None) == SHAPE
    assert "more than the kernel counts" in H.last_error()


@pytest.mark.parametrize("change,code", [
    ({"type": 0}, TYPE), ({"type": 3}, TYPE), ({"out_type": 3}, TYPE), ({"head_dim": 80}, SHAPE),
    ({"head_count": 5}, HEADS), ({"head_count_kv": 0}, HEADS), ({"scale": INF}, ARG), ({"scale": -0.5}, ARG),
    ({"sliding_window": -3}, ARG), ({"sequence_count": -1}, SHAPE), ({"sequence_count": (1 << 20) + 1}, SHAPE),
    ({"token_count": (1 << 30) + 1}, SHAPE), ({"q_stride": 255}, SHAPE), ({"k_stride": 132}, ARG),
    ({"v_stride": 100}, SHAPE), ({"k_stride": 1 << 24}, SHAPE), ({"output_stride": 260}, ARG), ({"d_q": None}, ARG), ({"d_offsets": None}, ARG),
    ({"d_k": P + 2}, ARG), ({"d_output": None}, ARG), ({"token_count": 1 << 30, "head_count": 65534}, SHAPE)])
def test_bad_packed(change, code):
    assert H.lib().hp_hip_packed_attention_device(packed(**change), None) == code


@pytest.mark.parametrize("change,code", [
    ({"rows": 65536}, SHAPE), ({"n": 0}, SHAPE), ({"n": (1 << 30) + 1}, SHAPE), ({"logits_stride": 99}, SHAPE),
    ({"output_stride": 99}, SHAPE), ({"allowed_stride": 3, "d_allowed": P}, SHAPE), ({"d_logits": None}, ARG),
    ({"d_output": None}, ARG), ({"d_history": P}, ARG), ({"d_history_lengths": P}, ARG), ({"d_bias_ids": P}, ARG),
    ({"d_bias_ids": P, "d_bias_values": P}, ARG), ({"d_bias_counts": P}, ARG), ({"history_stride": 1 << 31}, SHAPE),
    ({"bias_stride": 1 << 31}, SHAPE), ({"output_stride": 104}, ARG), ({"d_logits": P + 2}, ARG),
    ({"output_stride": 1 << 33}, SHAPE)])
def test_bad_rules(change, code):
    assert H.lib().hp_hip_logit_rules_device(rules(**change), None) == code


def test_null_structures_and_per_thread_stream():
    L = H.lib()
    assert L.hp_hip_paged_append_device(None, append(), None) == ARG
    assert L.hp_hip_paged_append_device(cache(), None, None) == ARG
    assert L.hp_hip_paged_attention_device(None, attention(), None) == ARG
    assert L.hp_hip_paged_attention_device(cache(), None, None) == ARG
    assert L.hp_hip_packed_attention_device(None, None) == ARG
    assert L.hp_hip_logit_rules_device(None, None) == ARG
    assert L.hp_hip_logit_rules_device(rules(), 2) == ARG  # hipStreamPerThread


def test_wrappers_raise():
    with pytest.raises(ValueError, match="paged_attention hip head count mismatch"):
        H.paged_attention_device(cache(), 3, P, 0, P, 0)
    with pytest.raises(TypeError, match="packed_attention hip unsupported type"):
        H.packed_attention_device(1, P, 1, 2, 2, 64, P, P, P, 0, P, 0)
    with pytest.raises(RuntimeError, match="logit_rules hip failed"):
        H.logit_rules_device(1, 10, 0, P)
    with pytest.raises(ValueError, match="paged_append hip shape mismatch"):
        H.paged_append_device(cache(), 7, 4, P, P, P, P, 1)


@pytest.mark.parametrize("scale", [3e38, 2.0 ** 121, INF])
def test_scales_whose_factors_are_no_numbers(scale):
    """scale * log2(e) and 1 / key_scale would be infinite, and a score or an element of 0 a NaN."""
    assert H.lib().hp_hip_paged_attention_device(cache(), attention(scale=scale), None) == ARG
    assert H.lib().hp_hip_packed_attention_device(packed(scale=scale), None) == ARG
    for name in ("key_scale", "value_scale"):
        for value in (scale, 1 / scale, 1e-39):
            c = cache(type=H.HP_ELEM_E4M3, **{name: value})
            assert H.lib().hp_hip_paged_append_device(c, append(), None) == ARG
            assert H.lib().hp_hip_paged_attention_device(c, attention(), None) == ARG
    c = cache(type=H.HP_ELEM_E4M3, key_scale=2.0 ** 100)
    assert H.lib().hp_hip_paged_attention_device(c, attention(scale=2.0 ** 21), None) == ARG
