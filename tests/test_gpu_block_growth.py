"""i8 blocks keep their scale, and what they hold, while elements as large as their largest come again."""
import numpy as np
import pytest

import test_gpu_long_context as base
from heliopause_amd import hip_kernels as H

pytestmark = pytest.mark.gpu


class Blocks:
    """One block of 16 positions for each of n sequences and two KV heads, filled a token at a time."""

    def __init__(self, n):
        t = base._torch()
        self.n, self.at = n, 0
        self.pools = [t.zeros((n, 2, 16, 64), dtype=t.int8, device="cuda") for _ in range(2)]
        self.scales = [t.full((n, 2, 1), float("nan"), device="cuda") for _ in range(2)]
        self.pages = base.dev(np.arange(n, dtype=np.int32)[:, None])

    def append(self, rows):
        """rows [n][2][64], as keys and as values."""
        self.at += 1
        length, d = base.dev(np.full(self.n, self.at, np.int32)), base.dev(rows)
        c = H.paged_cache(base.ptr(self.pools[0]), base.ptr(self.pools[1]), H.HP_ELEM_I8, page_count=self.n, page_size=16,
                          head_count_kv=2, head_dim=64, d_pages=base.ptr(self.pages), d_lengths=base.ptr(length),
                          sequence_count=self.n, pages_per_sequence=1)
        b = H.cache_blocks(16, d_key_scales=base.ptr(self.scales[0]), d_value_scales=base.ptr(self.scales[1]))
        H.block_append_device(c, b, self.n, 0, 0, base.ptr(d), 0, 0, 0)
        base.sync()
        assert base._torch().equal(self.scales[0], self.scales[1]) and base._torch().equal(*self.pools)
        return self.scales[0].cpu().numpy()[..., 0], self.pools[0].cpu().numpy()


def test_an_element_as_large_as_the_largest_does_not_grow_a_block(hip):
    rng = np.random.default_rng(1)
    x = (rng.standard_normal((1024, 2, 64)) * np.exp(rng.uniform(-40, 40, (1024, 2, 1)))).astype(np.float32)
    blocks = Blocks(1024)
    first, held = blocks.append(x)
    held = held[:, :, 0].copy()
    most = np.abs(x.astype(np.float64)).max(2)
    assert (np.abs(first * 127.0 - most) <= most * 3 * base.U).all()
    for row in (x, -x, x[..., ::-1].copy()):
        scales, stored = blocks.append(row)
        assert np.array_equal(scales, first)
    assert np.array_equal(stored[:, :, 0], held) and np.array_equal(stored[:, :, 1], held)
    assert np.array_equal(stored[:, :, 2], -held) and np.array_equal(stored[:, :, 3], held[..., ::-1])
    # the largest is 127 of its steps
    assert (np.abs(held).max(2) == 127).all()


def test_a_larger_element_does(hip):
    rng = np.random.default_rng(2)
    x = rng.standard_normal((64, 2, 64)).astype(np.float32)
    blocks = Blocks(64)
    first, _ = blocks.append(x)
    scales, _ = blocks.append((x * np.float32(1 + 2.0 ** -18)).astype(np.float32))
    assert (np.abs(scales / first.astype(np.float64) - 1.25) <= 1e-6).all()
