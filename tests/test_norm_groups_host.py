"""How many rows of the norms' gradients a group of lanes takes, read from the workspace (two sums of D a group)."""
import pytest

from tab_amd import _capi


def _groups(M, D, gates):
    size, rest = divmod(_capi.load().tab_norm_residual_backward_workspace_bytes(M, D, gates), 2 * D * 4)
    assert rest == 0
    return size


@pytest.mark.parametrize("M", [513, 514, 777, 778, 1001, 1531, 2047, 2048])
@pytest.mark.parametrize("gate_per_row", [False, True])
def test_two_rows_a_group_while_the_chip_holds_as_many(M, gate_per_row):
    """Rows of 1531 are held 1024 at once: half as many groups as rows, rounded up, for odd and even numbers of rows alike."""
    assert _groups(M, 1531, M if gate_per_row else 0) == (M + 1) // 2


def test_no_more_groups_than_the_chip_has_units_before_that_and_none_than_it_holds_after():
    assert [_groups(M, 1531, 0) for M in (1, 2, 255, 256, 257, 511, 512)] == [1, 2, 255, 256, 129, 256, 256]
    assert _groups(3000, 1531, 0) == 1000 and _groups(100000, 1531, 0) <= 1024
