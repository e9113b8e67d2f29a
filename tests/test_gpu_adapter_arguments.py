"""Numbers of groups that a C int does not hold."""
import pytest
import torch

from symmetrix_b200 import RowRouting

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("groups", [2 ** 32 + 3, -2 ** 32 + 3, 2 ** 64 + 3, 2 ** 31])
def test_numbers_of_groups_beyond_32_bits_are_refused(groups):
    with pytest.raises(ValueError, match="limits"):
        RowRouting(torch.zeros(4, dtype=torch.int32, device="cuda"), groups)
