"""When an i8 block grows, by the plain form (oracle/long_context.py).  CPU only."""
import numpy as np

from oracle import long_context as L


def test_a_scale_of_f32_holds_the_element_that_set_it():
    """f32's product of the largest element and 1 / 127 is up to 2^-23 below the quotient."""
    rng = np.random.default_rng(3)
    below = 0
    for most in np.exp(rng.uniform(-60, 60, 2000)).astype(np.float32):
        s = most * np.float32(1.0 / 127.0)
        below += float(s) * 127.0 < float(most)
        assert L.grown_scale("i8", float(s), float(most)) == float(s)
        assert L.grown_scale("i8", float(s), float(most) * (1 + 2.0 ** -18)) >= 1.25 * float(s)
        assert round(float(most) * float(np.float32(1.0) / s)) == 127
    assert below > 50


def test_e4m3_scales_have_no_slack():
    assert L.grown_scale("e4m3", 2.0 ** -3, 448.0 / 8) == 2.0 ** -3
    assert L.grown_scale("e4m3", 2.0 ** -3, np.nextafter(448.0 / 8, 100.0)) == 2.0 ** -2
