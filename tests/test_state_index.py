"""CPU: the row numbers that reorder_states and select_states take as sequences are whole numbers."""
import numpy as np
import pytest
import torch


@pytest.mark.parametrize("index", [[0.5, 1.0], [1.0, 0.0], [True, False], np.array([0.9, 1.2]), np.array([True, False]),
                                   (0.0,), np.zeros((2, 2)), float("nan")])
@pytest.mark.parametrize("name", ["reorder_states", "select_states"])
def test_other_numbers_are_refused(name, index):
    import burn_gdn2 as bg

    with pytest.raises(ValueError, match="whole numbers"):
        getattr(bg, name)(torch.zeros(2, 3), index)


@pytest.mark.parametrize("index,want", [([1, 0], [1, 0]), ((), []), ([], []), (np.array([1, -1], dtype=np.int32), [1, -1]),
                                        (np.array([], dtype=np.int64), []), (range(3), [0, 1, 2]), (np.uint8([2, 0]), [2, 0])])
def test_whole_numbers(index, want):
    from burn_gdn2 import sequence

    t = sequence._index("op", index)
    assert t.dtype == torch.int64 and t.tolist() == want
    given = torch.tensor([1], dtype=torch.int32)
    assert sequence._index("op", given) is given
