"""CPU checks of the bins that sample_tokens counts weights in (csrc/sample_bins.h, through the probe library; no GPU
call): a higher logit's bin is never lower, and every index that is made of bins stays within its array, whatever the
temperature and the logits."""
import ctypes
import itertools
import math
from pathlib import Path

import pytest
import torch

PROBE = Path(__file__).resolve().parents[1] / "llm-inference-optimizer_amd" / "libmi355_probe.so"
BINS = 256
MOST = torch.finfo(torch.float32).max
TEMPERATURES = [1e-45, 1e-40, 1.1754944e-38, 1e-30, 1e-3, 0.05, 0.7, 1.0, 100.0, 1e20, 1e30, 3e38, MOST, math.inf]
LOGITS = [-MOST, -1e30, -1e10, -65504.0, -37.5, -1.0, -1e-3, -1e-30, -1e-45, -0.0, 0.0, 1e-45, 1e-30, 1e-3, 1.0, 3.0, 37.5,
          65504.0, 1e10, 1e30, MOST, math.inf]


@pytest.fixture(scope="module")
def bins():
    if not PROBE.exists():
        pytest.skip("probe library not built")
    f = ctypes.CDLL(str(PROBE)).mi355_probe_sample_bins
    f.argtypes, f.restype = [ctypes.c_float] * 4 + [ctypes.POINTER(ctypes.c_int)], None

    def call(temperature, x, part, row):
        out = (ctypes.c_int * 3)()
        f(temperature, x, part, row, out)
        return tuple(out)
    return call


@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_bins_are_monotone(bins, temperature):
    of = [bins(temperature, x, x, x)[0] for x in LOGITS]
    assert of == sorted(of)
    # infinity is no finite logit's bin where those have one bin together
    assert temperature < math.inf or (len(set(of[:-1])) == 1 and of[-1] - of[0] >= BINS)


@pytest.mark.parametrize("temperature", TEMPERATURES)
def test_indexes_stay_within_the_bins(bins, temperature):
    for x, part, row in itertools.combinations_with_replacement(LOGITS, 3):
        _, at, shift = bins(temperature, x, part, row)
        assert 0 <= at < BINS, (x, part, row)
        assert 0 <= shift <= BINS, (x, part, row)  # the kernel reads bin max(g - shift, 0) for g < 256
