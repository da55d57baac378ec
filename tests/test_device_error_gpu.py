"""Who reads the library's device error word, and when."""

from __future__ import annotations

import pytest
import torch

from src import _native as nat

pytestmark = pytest.mark.gpu


def test_reading_waits_for_streams_of_their_own():
    """PyTorch's streams do not block the legacy stream: a wait that runs out
    on one of them is still seen by the next read."""
    assert nat.device_error(reset=True) == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # some 50 ms
        assert nat.load().m3_selftest_wait_timeout(side.cuda_stream) == nat.M3_OK
    assert nat.device_error(reset=True) == nat.M3_DEVERR_TIMEOUT
    assert nat.device_error() == 0
