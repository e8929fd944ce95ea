r"""Layers for wide networks where no GPU is needed: argument errors of the C entry points and of the Python functions."""
import pytest
import torch

from triton_helpers_b200 import _lib, build
from triton_helpers_b200.layers.checkpointed_linear import CheckpointedLinear, checkpointed_linear
from triton_helpers_b200.layers.int8_linear import Int8Rows, dequantize_rows, int8_linear, quantize_rows
from triton_helpers_b200.layers.rms_norm import RMSNorm, rms_norm, rms_norm_int8

AT = 1 << 20  # an aligned address that no call here gets to read


@pytest.fixture(scope="module")
def library():
    if not _lib.LIB_PATH.exists():
        build.build()
    return _lib.lib()


def said(library, text):
    return text in library.th_last_error_string()


def test_rows_entry_points_refuse(library):
    assert library.th_rms_norm_fwd(AT, 8, None, 0, AT, 0, None, AT, None, -1, 8, 1e-6, 0, None) == -1
    assert library.th_rms_norm_fwd(AT, 8, None, 0, AT, 0, None, AT, None, 4, 0, 1e-6, 0, None) == -1
    assert library.th_rms_norm_fwd(AT, 8, None, 0, AT, 0, None, AT, None, 4, 8, 1e-6, 7, None) == -2 and said(library, b"dtype")
    assert library.th_rms_norm_fwd(AT, 8, None, 0, AT, 2, None, AT, None, 4, 8, 1e-6, 1, None) == -2 and said(library, b"gain")
    assert library.th_rms_norm_fwd(AT, 8, AT, 8, AT, 0, None, AT, None, 4, 8, 1e-6, 0, None) == -1 and said(library, b"null")  # residual without sum
    assert library.th_rms_norm_fwd(None, 8, None, 0, AT, 0, None, AT, None, 0, 8, 1e-6, 0, None) == 0  # no rows
    assert library.th_rms_norm_fwd(AT + 2, 8, None, 0, AT, 0, None, AT, None, 4, 8, 1e-6, 0, None) == -3 and said(library, b"elements")
    assert library.th_rms_norm_int8(AT, 8, None, 0, AT, 0, None, AT, 8, AT, 4, 8, 1e-6, 0, None) == -3 and said(library, b"16 bytes")
    assert library.th_quantize_rows(AT, 8, AT + 8, 16, AT, 4, 8, 0, None) == -3
    assert library.th_quantize_rows(AT, 40, AT, 32, AT, 4, 40, 0, None) == -3  # rows longer than their stride
    assert library.th_quantize_rows(AT, 8, AT, 1 << 25, AT, 4, (1 << 24) + 1, 0, None) == -2
    assert library.th_dequantize_rows(AT, 8, AT, AT, 7, 4, 8, 0, None) == -1
    assert library.th_rms_norm_bwd(AT, 8, AT, 0, AT, AT, 8, None, 0, AT, AT, None, 0, 4, 8, 0, None) == -4 and said(library, b"scratch")
    assert library.th_column_sum(AT, 8, AT, None, 0, 4, 8, 0, None) == -4
    assert library.th_checkpoint_rows(AT, 16, AT, AT, 8, 8, AT, 8, AT, 8, None, 0, 4, 1, None) == -4
    assert library.th_checkpoint_rows(AT, 16, AT, AT, 8, 8, AT, 8, AT, 8, AT, 1 << 20, 4, 0, None) == -2


def test_product_entry_points_refuse(library):
    assert library.th_int8_linear(AT, 16, AT, AT, 16, AT, None, AT, 8, 4, 131072, 8, 0, None) == -2 and said(library, b"32-bit")
    assert library.th_int8_linear(AT, 24, AT, AT, 16, AT, None, AT, 8, 4, 16, 8, 0, None) == -3
    assert library.th_int8_linear(AT, 16, AT, AT + 4, 16, AT, None, AT, 8, 4, 16, 8, 0, None) == -3
    assert library.th_int8_linear(AT, 16, None, AT, 16, AT, None, AT, 8, 4, 16, 8, 0, None) == -1
    assert library.th_int8_linear(AT, 16, AT, AT, 16, AT, None, AT, 7, 4, 16, 8, 0, None) == -1
    assert library.th_int8_linear(AT, 16, AT, AT, 16, AT, None, AT, 8, 4, 16, 8, 5, None) == -2
    assert library.th_int8_linear(None, 16, None, None, 16, None, None, None, 8, 0, 16, 8, 0, None) == 0
    assert library.th_linear_fwd(AT, 16, AT, 16, None, AT, 8, 4, 16, 8, 0, None) == -2 and said(library, b"float16")
    assert library.th_linear_fwd(AT, 15, AT, 16, None, AT, 8, 4, 16, 8, 1, None) == -1
    assert library.th_linear_fwd(AT, 16, AT, 16, None, AT, 8, -4, 16, 8, 1, None) == -1
    assert library.th_linear_bwd_input(AT, 7, AT, 16, AT, 16, 4, 16, 8, 1, None) == -1
    assert library.th_linear_bwd_weight(AT, 8, AT, 16, None, 4, 16, 8, 1, None) == -1
    assert library.th_linear_fwd(AT, 16, AT, 16, None, AT, 8, (1 << 30) + 1, 16, 8, 1, None) == -2


def test_scratch_sizes(library):
    for rows, d, dtype in ((1, 1, 0), (7, 33, 1), (4096, 4096, 2), (3, 100000, 0), (100000, 16, 1)):
        assert library.th_rms_norm_bwd_workspace_bytes(rows, d, dtype) >= 4 * d
        assert library.th_column_sum_workspace_bytes(rows, d) >= 4 * d
    assert library.th_rms_norm_bwd_workspace_bytes(0, 8, 0) == 0 and library.th_column_sum_workspace_bytes(0, 8) == 0


def test_python_functions_refuse():
    x, gain = torch.randn(4, 32), torch.ones(32)
    with pytest.raises(AssertionError, match="same device"):
        rms_norm(x, gain)
    with pytest.raises(AssertionError, match="same device"):
        quantize_rows(x)
    with pytest.raises(AssertionError, match="same device"):
        checkpointed_linear(x.half(), torch.randn(8, 32).half())
    with pytest.raises(AssertionError, match="Weight shape"):
        rms_norm(x, torch.ones(31))
    with pytest.raises(AssertionError, match="Residual"):
        rms_norm(x, gain, x[:1])
    with pytest.raises(TypeError):
        rms_norm(x.int(), gain)
    with pytest.raises(TypeError):
        rms_norm(x, gain.half())
    with pytest.raises(AssertionError):
        rms_norm(x[:, :0], gain[:0])
    with pytest.raises(RuntimeError, match="no gradient"):
        rms_norm_int8(x, gain.requires_grad_(True))
    with pytest.raises(TypeError):
        checkpointed_linear(x, torch.randn(8, 32))
    with pytest.raises(AssertionError, match="Input dimension"):
        checkpointed_linear(x.half(), torch.randn(8, 31).half())
    rows = Int8Rows(torch.zeros(4, 32, dtype=torch.int8), torch.ones(4))
    with pytest.raises(TypeError, match="dtype"):
        int8_linear(rows, rows)
    with pytest.raises(TypeError, match="int8"):
        int8_linear(rows, Int8Rows(rows.q.int(), rows.scale), dtype=torch.float32)
    with pytest.raises(AssertionError, match="one scale per row"):
        int8_linear(rows, Int8Rows(rows.q, rows.scale[:3]), dtype=torch.float32)
    with pytest.raises(AssertionError, match="matrix"):
        int8_linear(rows, Int8Rows(rows.q[None], rows.scale[None]), dtype=torch.float32)
    with pytest.raises(AssertionError, match="same device"):
        dequantize_rows(rows)


def test_modules_have_the_parameters_of_their_plain_forms():
    plain, layer = torch.nn.Linear(48, 24), CheckpointedLinear(48, 24)
    layer.load_state_dict(plain.state_dict())
    assert torch.equal(layer.weight, plain.weight) and torch.equal(layer.bias, plain.bias)
    assert RMSNorm(16).state_dict().keys() == {"weight"} and torch.equal(RMSNorm(16).weight, torch.ones(16))
