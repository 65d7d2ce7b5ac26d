"""The polynomial that the 8-bit product's gelu is computed with, as it stands in the source, against erfc in 64 bits."""
import math
import re

import torch

from tensor_parallel_b200 import build


def _polynomial():
    source = (build.CSRC / "gemm_i8.cuh").read_text()
    comment, body = re.search(r"((?://[^\n]*\n)+)__device__ __forceinline__ float i8_gelu\(float v\) \{(.*?)\n\}", source, re.S).groups()
    slope = float(re.search(r"__fmaf_rn\((\S+)f, fabsf\(v\), 1\.f\)", body).group(1))
    coefficients = [float(re.search(r"float s = (\S+)f;", body).group(1))] + [float(c) for c in re.findall(r"s = __fmaf_rn\(s, t, (\S+)f\);", body)]
    as_stored = [torch.tensor(c, dtype=torch.float32).item() for c in (slope, *coefficients)]
    return as_stored[0], as_stored[1:], " ".join(comment.replace("//", " ").split())


def test_the_error_is_what_the_source_says():
    slope, coefficients, comment = _polynomial()
    assert len(coefficients) == 7
    v = torch.linspace(0, 14, 1400001, dtype=torch.float64)
    t, s = 1 / (1 + slope * v), torch.zeros_like(v)
    for c in coefficients:
        s = s * t + c
    half = 0.5 * torch.special.erfc(v / math.sqrt(2))
    off = (s * t * torch.exp(-v * v / 2) - half).abs()
    said = re.search(r"half of erfc is off by (\S+) \((\S+) of it up to v = 5, (\S+) up to 8, (\S+) up to 13\), v times it by (\S+);", comment).groups()
    found = [off.max(), *((off / half)[v <= end].max() for end in (5, 8, 13)), (v * off).max()]
    for bound, value in zip(map(float, said), found):
        assert 0.9 * bound <= value <= bound
    # what is left of a tail's value after the rounding to bf16 (2^-9 of it at most) is no worse for it
    assert found[3] < 2.0 ** -9
