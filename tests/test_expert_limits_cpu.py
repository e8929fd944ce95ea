r"""Layers of experts: sizes whose rows 32 bits cannot count are refused before anything is launched."""
import pytest

from triton_helpers_b200 import _lib, build

AT = 1 << 20  # an aligned address that no call here gets to read


@pytest.mark.parametrize("experts,d_out", [(131, 16393004), (129, 16647160), (128, 1 << 24), (1024, 1 << 21)])
def test_gradients_of_too_many_rows_are_refused(experts, d_out):
    # 131 x 16393004 rows are below 2^31; the last tile's, which are counted too, are not
    if not _lib.LIB_PATH.exists():
        build.build()
    library = _lib.lib()
    assert library.th_expert_linear_bwd_weight(AT, -(-d_out // 8) * 8, AT, 8, AT, AT, 4, experts, 8, d_out, 1, None) == -2
    assert b"experts" in library.th_last_error_string()
