"""What packed_plan takes as lengths (CPU)."""
import numpy as np
import pytest
import torch

import cudatransformer_amd as ct


@pytest.mark.parametrize("lens", [[3, 0, 5], (3, 0, 5), np.array([3, 0, 5]), torch.tensor([3, 0, 5], dtype=torch.int32),
                                  [np.int64(3), torch.tensor(0), 5]])
def test_whole_numbers(lens):
    assert ct.packed_plan(lens, 2, 2, device="cpu").seqlens == (3, 0, 5)


@pytest.mark.parametrize("lens", [[3.0], [3.7, 2], np.array([3.5]), [torch.tensor(2.5)], ["3"], [None], 5])
def test_others_are_refused(lens):
    with pytest.raises(ValueError):
        ct.packed_plan(lens, 2, 2, device="cpu")
