"""CPU: how many batches are in flight by default follows the hardware queues of the process."""
import pytest

from dnascent_amd import hip


@pytest.mark.parametrize("queues,network,banded", [(None, 6, 8), ("8", 6, 8), ("16", 6, 8), ("7", 4, 7), ("6", 4, 6), ("5", 3, 5), ("4", 3, 4), ("2", 3, 2), ("1", 3, 1), ("x", 3, 4)])
def test_batches_in_flight(monkeypatch, queues, network, banded):
    if queues is None:
        monkeypatch.delenv("GPU_MAX_HW_QUEUES", raising=False)
    else:
        monkeypatch.setenv("GPU_MAX_HW_QUEUES", queues)
    assert hip.batches_in_flight(6) == network and hip.batches_in_flight(8, network=False) == banded
    assert hip.batches_in_flight(2) == 2 and hip.batches_in_flight(1, network=False) == 1
