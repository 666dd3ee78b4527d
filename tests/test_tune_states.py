"""What AdamW and Adapters make of their surroundings and of what they are given, without a GPU: tensors that say that
they are on one, and entries that count their calls (as in test_tune.py)."""
import pytest

torch = pytest.importorskip("torch")

from ytm_amd import tune  # noqa: E402

from test_tune import entries, on_gpu  # noqa: E402, F401


def test_tables_are_made_on_the_host(entries):  # noqa: F811
    p, g = on_gpu(300), on_gpu(300)
    with torch.device("meta"):
        a = tune.AdamW([p], [g])
    assert a._table.device.type == "cpu"
