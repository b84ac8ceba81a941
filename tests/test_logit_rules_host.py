"""What ``LogitRules`` takes as a mask (no GPU needed: the struct that the call gets)."""
import pytest
import torch

from oxinfer_b200.sampling import LogitRules

CPU = torch.device("cpu")


@pytest.mark.parametrize("t,n,shape,stride", [(3, 100, (4,), 0), (3, 100, (1, 4), 0), (3, 100, (3, 4), 4), (3, 100, (1, 9), 0), (3, 100, (3, 9), 9), (1, 100, (4,), 4), (1, 100, (9,), 9),
                                              (1, 128, (1, 4), 4), (3, 129, (5,), 0)])
def test_masks_of_one_row_and_of_all(t, n, shape, stride):
    mask = torch.zeros(shape, dtype=torch.int32)
    r = LogitRules(mask=mask).c(t, n, CPU)
    assert r.mask == mask.data_ptr() and (r.mask_stride == stride or t == 1)


@pytest.mark.parametrize("t,n,shape", [(3, 100, (12,)), (3, 100, (5,)), (3, 100, (3,)), (3, 100, (2, 4)), (3, 100, (3, 3)), (2, 64, (4,)), (3, 100, ())])
def test_masks_that_are_refused(t, n, shape):
    """A flat mask of all rows is none of one row for all."""
    with pytest.raises(AssertionError):
        LogitRules(mask=torch.zeros(shape, dtype=torch.int32)).c(t, n, CPU)
