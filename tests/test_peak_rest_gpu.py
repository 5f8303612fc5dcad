"""The measured tensor rate does not go with what ran before it: every measurement starts from rest."""
import time

import pytest

import fenix_b200 as fx

pytestmark = pytest.mark.gpu


def test_rate_after_other_work(cuda_torch):
    rates = []
    for _ in range(4):
        time.sleep(0.5)
        rates.append(fx.tc_peak("f16", 20.0, 3)[0])  # the GPU is at rest
        fx.tc_peak("fp8", 60.0, 3)  # long enough for the power limit to act
        rates.append(fx.tc_peak("f16", 20.0, 3)[0])  # it was not
    print("f16 rates at rest and after e4m3 runs:", [round(r) for r in rates])
    # one clock for all of them; held down by the power limit the latter were up to a fifth lower
    assert max(rates) / min(rates) < 1.1
