"""The scored attention's tanh, its polynomial as the source has it, against tanh in 64 bits."""
import os
import re

import numpy as np

from rtp_llm_amd import build


def test_polynomial_is_as_near_as_its_comment_says():
    src = open(os.path.join(build.CSRC, "scored.h")).read()
    body = src[src.index("float tanh_near"):src.index("float tanh_far")]
    near = float(re.search(r"kTanhNear = ([0-9.]+)f", src).group(1))
    said = float(re.search(r"([0-9.]+e-9) relative", src).group(1))
    c = [float(np.float32(x)) for x in [re.search(r"float r = (-?[0-9.]+)f", body).group(1)] + re.findall(r"__builtin_fmaf\(r, z, (-?[0-9.]+)f\)", body)]
    assert len(c) == 5
    u = np.linspace(1e-3, near, 400001)
    z, r = u * u, 0.0
    for x in c:
        r = r * z + x
    worst = float(np.abs((u + u * z * r) / np.tanh(u) - 1).max())
    assert 0.98 * said <= worst <= said, worst
