"""Argument checks and index rules of the operators of long contexts (page plans, pages with block scales, block bounds,
selection and attention).  CPU only: every call here is refused on the host before a device is looked for."""
import shutil
import subprocess
from pathlib import Path

import pytest

from heliopause_amd import hip_kernels as H

ROOT = Path(__file__).resolve().parents[1]
P = 1 << 20  # a 16-byte aligned address that no call gets as far as reading
NAN, INF = float("nan"), float("inf")
SHAPE, HEADS, TYPE, ARG = H.HP_ERR_SHAPE, H.HP_ERR_HEADS, H.HP_ERR_TYPE, H.HP_ERR_ARG


def test_index_rules(tmp_path):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "long_index"
    subprocess.run([cxx, "-std=c++17", "-O1", "-Wall", "-Werror", str(ROOT / "tests" / "long_index.cpp"), "-o", str(exe)],
                   check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout + r.stderr


def changed(p, change):
    for name, value in change.items():
        setattr(p, name, value)
    return p


def cache(**change):
    return changed(H.paged_cache(P, P, H.HP_ELEM_I8, page_count=4, page_size=32, head_count_kv=2, head_dim=64, d_pages=P,
                                 d_lengths=P, sequence_count=3, pages_per_sequence=2), change)


def blocks(**change):
    return changed(H.cache_blocks(16, d_key_scales=P, d_value_scales=P, d_key_bounds=P), change)


def append(**change):
    return changed(H.HipPagedAppend(d_q=P, d_k=P, d_v=P, d_q_out=P, token_count=3, head_count=4, out_type=H.HP_ELEM_F16,
                                    rope_dims=64, rope_freq_base=1e4, epsilon=1e-6), change)


def attention(**change):
    return changed(H.HipPagedAttention(d_q=P, d_output=P, head_count=4, q_type=H.HP_ELEM_F32, out_type=H.HP_ELEM_F32,
                                       scale=1.0), change)


def select(**change):
    return changed(H.HipBlockSelect(d_q=P, d_selected=P, d_counts=P, head_count=4, q_type=H.HP_ELEM_F32, budget=4,
                                    first_blocks=1, last_blocks=1), change)


def plan(**change):
    return changed(H.HipPagePlan(d_pages=P, d_lengths=P, d_new_tokens=P, d_lengths_out=P, d_free=P, d_free_count=P, d_slots=P,
                                 token_count=9, sequence_count=3, pages_per_sequence=4, page_size=16, page_count=10), change)


def calls(c, b):
    L = H.lib()
    return [L.hp_hip_block_append_device(c, b, append(), None), L.hp_hip_block_bounds_device(c, b, None, 3, None),
            L.hp_hip_block_select_device(c, b, select(), None),
            L.hp_hip_block_attention_device(c, b, attention(), P, P, 4, None)]


@pytest.mark.parametrize("change,code", [
    ({"type": 0}, TYPE), ({"type": 5}, TYPE), ({"type": -1}, TYPE), ({"head_dim": 96}, SHAPE), ({"head_count_kv": 0}, HEADS),
    ({"page_size": 8}, SHAPE), ({"page_size": 48}, SHAPE), ({"page_count": 0}, SHAPE), ({"sequence_count": -1}, SHAPE),
    ({"pages_per_sequence": 0}, SHAPE), ({"page_stride": 4095}, SHAPE), ({"page_stride": 4104}, ARG), ({"d_keys": None}, ARG),
    ({"d_pages": None}, ARG), ({"d_lengths": None}, ARG), ({"d_values": P + 8}, ARG)])
def test_bad_caches(change, code):
    assert calls(cache(**change), blocks()) == [code] * 4


@pytest.mark.parametrize("change,code", [
    ({"block_size": 8}, SHAPE), ({"block_size": 0}, SHAPE), ({"block_size": 24}, SHAPE), ({"block_size": 64}, SHAPE),
    ({"block_size": -16}, SHAPE), ({"reserved": 1}, ARG), ({"d_key_scales": None}, ARG), ({"d_value_scales": None}, ARG),
    ({"d_key_scales": None, "d_value_scales": None}, ARG), ({"d_key_scales": P + 2}, ARG), ({"d_key_bounds": P + 8}, ARG)])
def test_bad_blocks(change, code):
    assert calls(cache(), blocks(**change)) == [code] * 4


def test_blocks_up_to_128():
    assert calls(cache(page_size=256), blocks(block_size=256)) == [SHAPE] * 4


def test_types_and_scales():
    L = H.lib()
    plain = blocks(d_key_scales=None, d_value_scales=None)
    for t in (H.HP_ELEM_F16, H.HP_ELEM_BF16):  # 16-bit pages have no scales
        assert calls(cache(type=t), blocks()) == [TYPE] * 4
        assert L.hp_hip_block_append_device(cache(type=t), plain, append(), None) == TYPE
        assert L.hp_hip_block_attention_device(cache(type=t), plain, attention(), None, None, 0, None) == ARG
    e4m3 = H.HP_ELEM_E4M3
    assert L.hp_hip_block_append_device(cache(type=e4m3), plain, append(), None) == ARG
    assert L.hp_hip_block_attention_device(cache(type=e4m3), plain, attention(), None, None, 0, None) == ARG
    # one scale of the whole cache counts only where the blocks have none
    for bad in (0.0, NAN, 2.0 ** 101):
        assert L.hp_hip_block_attention_device(cache(type=e4m3, key_scale=bad), plain, attention(), P, P, 4, None) == ARG
        assert L.hp_hip_block_attention_device(cache(type=e4m3, key_scale=bad), blocks(), attention(scale=0.0), P, P, 4, None) == ARG
        assert "scale (times" in H.last_error()
    # i8 pages are these entry points' alone
    assert L.hp_hip_paged_append_device(cache(), append(), None) == TYPE
    assert L.hp_hip_paged_attention_device(cache(), attention(), None) == TYPE


@pytest.mark.parametrize("change,code", [
    ({"out_type": 3}, TYPE), ({"out_type": 4}, TYPE), ({"head_count": 3}, HEADS), ({"head_count": 0}, HEADS), ({"d_q": None}, ARG),
    ({"d_q_out": None}, ARG), ({"d_k": None}, ARG), ({"rope_dims": 12}, SHAPE), ({"rope_dims": 72}, SHAPE),
    ({"rope_freq_base": NAN}, ARG), ({"epsilon": -1.0}, ARG), ({"token_count": 2}, SHAPE),
    ({"token_count": (1 << 23) + 1, "d_offsets": P}, SHAPE), ({"q_stride": 258}, ARG), ({"k_stride": 127}, SHAPE),
    ({"d_v": P + 8}, ARG), ({"d_k_out": P + 4}, ARG)])
def test_bad_appends(change, code):
    assert H.lib().hp_hip_block_append_device(cache(), blocks(), append(**change), None) == code


def test_more_rows_than_a_launch_takes():
    big = append(token_count=1 << 23, d_offsets=P, head_count=1024)
    assert H.lib().hp_hip_block_append_device(cache(), blocks(), big, None) == SHAPE
    c = cache(head_count_kv=65535, sequence_count=65535)
    assert H.lib().hp_hip_block_bounds_device(c, blocks(), None, 65535, None) == SHAPE
    c = cache(sequence_count=65535, pages_per_sequence=1 << 25)
    assert H.lib().hp_hip_block_select_device(c, blocks(), select(), None) == SHAPE
    c = cache(sequence_count=65535, head_count_kv=4)
    assert H.lib().hp_hip_block_attention_device(c, blocks(block_size=32), attention(), P, P, 1 << 20, None) == SHAPE
    assert "more than the kernel counts" in H.last_error()


def test_bad_bounds():
    L = H.lib()
    assert L.hp_hip_block_bounds_device(cache(), blocks(), None, 2, None) == SHAPE
    assert L.hp_hip_block_bounds_device(cache(), blocks(), P, (1 << 23) + 1, None) == SHAPE
    assert L.hp_hip_block_bounds_device(cache(), blocks(d_key_bounds=None), None, 3, None) == ARG


@pytest.mark.parametrize("change,code", [
    ({"head_count": 3}, HEADS), ({"head_count": 0}, HEADS), ({"q_type": 3}, TYPE), ({"q_type": 4}, TYPE), ({"budget": 0}, SHAPE),
    ({"budget": -1}, SHAPE), ({"budget": (1 << 20) + 1}, SHAPE), ({"first_blocks": -1}, SHAPE), ({"last_blocks": -1}, SHAPE),
    ({"first_blocks": 3, "last_blocks": 2}, SHAPE), ({"first_blocks": 2147483647, "last_blocks": 2147483647}, SHAPE),
    ({"reserved": 7}, ARG), ({"q_stride": 255}, SHAPE), ({"q_stride": 257}, ARG), ({"d_q": None}, ARG),
    ({"d_selected": None}, ARG), ({"d_q": P + 4}, ARG)])
def test_bad_selections(change, code):
    assert H.lib().hp_hip_block_select_device(cache(), blocks(), select(**change), None) == code


def test_selection_needs_bounds():
    assert H.lib().hp_hip_block_select_device(cache(), blocks(d_key_bounds=None), select(), None) == ARG


@pytest.mark.parametrize("change,code", [
    ({"head_count": 3}, HEADS), ({"head_count": 65536}, HEADS), ({"q_type": 3}, TYPE), ({"out_type": -1}, TYPE),
    ({"scale": 0.0}, ARG), ({"scale": NAN}, ARG), ({"scale": 2.0 ** 121}, ARG), ({"sliding_window": -1}, ARG),
    ({"reserved": 1}, ARG), ({"q_stride": 128}, SHAPE), ({"output_stride": 257}, ARG), ({"d_q": None}, ARG), ({"d_output": P + 4}, ARG)])
@pytest.mark.parametrize("selected", [False, True])
def test_bad_attentions(change, code, selected):
    listed = (P, P, 4) if selected else (None, None, 0)
    assert H.lib().hp_hip_block_attention_device(cache(), blocks(), attention(**change), *listed, None) == code


def test_bad_lists():
    L = H.lib()
    f = lambda *a, **change: L.hp_hip_block_attention_device(cache(), blocks(), attention(**change), *a, None)  # noqa: E731
    assert f(P, P, 0) == SHAPE and f(P, P, -1) == SHAPE and f(P, P, (1 << 20) + 1) == SHAPE
    assert f(None, P, 0) == ARG and f(None, None, 4) == ARG
    assert f(P, P, 4, sliding_window=100) == ARG


@pytest.mark.parametrize("change,code", [
    ({"sequence_count": -1}, SHAPE), ({"sequence_count": 65536}, SHAPE), ({"page_size": 8}, SHAPE), ({"page_size": 40}, SHAPE),
    ({"page_size": 8192}, SHAPE), ({"page_count": 0}, SHAPE), ({"pages_per_sequence": 0}, SHAPE),
    ({"pages_per_sequence": (1 << 26) + 1}, SHAPE), ({"sequence_count": 65535, "pages_per_sequence": 1 << 16}, SHAPE),
    ({"token_count": (1 << 30) + 1}, SHAPE), ({"d_new_tokens": None, "token_count": 4}, SHAPE), ({"d_pages": None}, ARG),
    ({"d_lengths": None}, ARG), ({"d_lengths_out": None}, ARG), ({"d_free": None}, ARG), ({"d_free_count": None}, ARG),
    ({"d_pages": P + 2}, ARG), ({"d_keep_from": P + 1}, ARG), ({"d_slots": P + 4}, ARG)])
def test_bad_plans(change, code):
    assert H.lib().hp_hip_page_plan_device(plan(**change), None) == code


def test_null_structures_and_per_thread_stream():
    L = H.lib()
    assert L.hp_hip_page_plan_device(None, None) == ARG
    assert L.hp_hip_page_plan_device(plan(), 2) == ARG  # hipStreamPerThread
    c, b = cache(), blocks()
    for x, y, z in ((None, b, True), (c, None, True), (c, b, False)):
        assert L.hp_hip_block_append_device(x, y, append() if z else None, None) == ARG
        assert L.hp_hip_block_select_device(x, y, select() if z else None, None) == ARG
        assert L.hp_hip_block_attention_device(x, y, attention() if z else None, P, P, 4, None) == ARG
    assert L.hp_hip_block_bounds_device(None, b, None, 3, None) == ARG
    assert L.hp_hip_block_bounds_device(c, None, None, 3, None) == ARG
    assert L.hp_hip_block_append_device(c, b, append(), 2) == ARG


def test_wrappers_raise():
    with pytest.raises(ValueError, match="block_attention hip head count mismatch"):
        H.block_attention_device(cache(), blocks(), 3, P, 0, P, 0)
    with pytest.raises(TypeError, match="block_append hip unsupported type"):
        H.block_append_device(cache(type=H.HP_ELEM_F16), blocks(d_key_scales=None, d_value_scales=None), 3, 4, P, P, P, P, 1)
    with pytest.raises(ValueError, match="block_select hip shape mismatch"):
        H.block_select_device(cache(), blocks(), 4, P, 0, 0, P)
    with pytest.raises(RuntimeError, match="page_plan hip failed"):
        H.page_plan_device(3, 4, 16, 10, 0, P, P, P, P)
    with pytest.raises(ValueError, match="block_bounds hip shape mismatch"):
        H.block_bounds_device(cache(), blocks(), 4)
