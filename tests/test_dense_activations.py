"""The normal tail's polynomials in the dense kernels: the constants as they stand
in the source, evaluated in 64 bits, against the tail itself."""

import os
import re

import numpy as np
import pytest
from scipy import special

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), 'vectra_amd', 'csrc', 'dense',
                      'dense_common.h')


def constants(which):
    """(c, coefficients from the highest power down) as the fp32 values they are."""
    with open(SOURCE, encoding='utf-8') as f:
        text = f.read()
    body = re.search(r'void normal_tail\(.*?\n}', text, re.S).group(0).split('} else {')[which]
    c = re.search(r'fmaf\((\S+)f, a, 1\.f\)', body).group(1)
    powers = [re.search(r'p = (-?\d\S*)f;', body).group(1), *re.findall(r'fmaf\(p, t, (-?\S+)f\)', body)]
    return float(np.float32(c)), [float(np.float32(v)) for v in powers]


# The figures that the source states, to their last digit.
@pytest.mark.parametrize('which,degree,bound', [(0, 8, 3.05e-8), (1, 6, 8.25e-7)], ids=['fp32', '16 bits'])
def test_the_tail_is_as_close_as_the_source_says(which, degree, bound):
    c, powers = constants(which)
    assert len(powers) == degree + 1
    a = np.linspace(0.0, 14.0, 400001)
    t = 1.0 / (1.0 + c * a)
    # Phi(-a) / exp(-a^2 / 2) = erfcx(a / sqrt(2)) / 2, which underflows nowhere.
    want = special.erfcx(a / np.sqrt(2.0)) / 2
    assert np.abs(np.polyval(powers, t) * t / want - 1.0).max() < bound
