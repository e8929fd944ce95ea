r"""Layers for wide networks where no GPU is needed: pointers that the C entry points refuse before they launch anything."""
import pytest

from triton_helpers_b200 import _lib, build

AT = 1 << 20  # an aligned address that no call here gets to read


@pytest.fixture(scope="module")
def library():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


# every pointer's place among the arguments, with the bytes of its element, in calls that are otherwise in order
CALLS = {
    "th_rms_norm_fwd": ((AT, 8, AT, 8, AT, 0, AT, AT, AT, 4, 8, 1e-6, 1, None), {0: 2, 2: 2, 4: 4, 6: 2, 7: 2, 8: 4}),
    "th_rms_norm_int8": ((AT, 8, AT, 8, AT, 1, AT, AT, 16, AT, 4, 8, 1e-6, 1, None), {0: 2, 2: 2, 4: 2, 6: 2, 9: 4}),
    "th_rms_norm_bwd": ((AT, 8, AT, 0, AT, AT, 8, AT, 8, AT, AT, AT, 1 << 20, 4, 8, 1, None), {0: 2, 2: 4, 4: 4, 5: 2, 7: 2, 9: 2, 10: 4}),
    "th_quantize_rows": ((AT, 8, AT, 16, AT, 4, 8, 0, None), {0: 4, 4: 4}),
    "th_dequantize_rows": ((AT, 16, AT, AT, 8, 4, 8, 2, None), {2: 4, 3: 2}),
    "th_column_sum": ((AT, 8, AT, AT, 1 << 20, 4, 8, 1, None), {0: 2, 2: 2}),
    "th_checkpoint_rows": ((AT, 16, AT, AT, 8, 8, AT, 8, AT, 8, AT, 1 << 20, 4, 1, None), {2: 4, 3: 2, 6: 2, 8: 2}),
    "th_int8_linear": ((AT, 16, AT, AT, 16, AT, AT, AT, 8, 4, 16, 8, 1, None), {2: 4, 5: 4, 6: 2, 7: 2}),
    "th_quantized_linear": ((AT, 16, 0, AT, 16, AT, AT, AT, 8, AT, 1 << 20, 4, 16, 8, 1, None), {0: 4, 5: 4, 6: 2, 7: 2}),
    "th_linear_fwd": ((AT, 16, AT, 16, AT, AT, 8, 4, 16, 8, 1, None), {4: 2, 5: 2}),
    "th_linear_bwd_input": ((AT, 8, AT, 16, AT, 16, 4, 16, 8, 1, None), {4: 2}),
    "th_linear_bwd_weight": ((AT, 8, AT, 16, AT, 4, 16, 8, 1, None), {4: 2}),
}


@pytest.mark.parametrize("name,place", [(name, place) for name, (_, places) in CALLS.items() for place in places])
def test_a_pointer_off_its_elements_is_refused(library, name, place):
    args, places = CALLS[name]
    off = [AT + places[place] // 2 if k == place else v for k, v in enumerate(args)]
    assert getattr(library, name)(*off) == -3 and b"elements" in library.th_last_error_string()
