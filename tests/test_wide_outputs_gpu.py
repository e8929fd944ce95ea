r"""Products into a part of a larger matrix, called through the C ABI: what lies beside the part stays as it was."""
import pytest
import torch

from triton_helpers_b200 import _lib
from triton_helpers_b200.layers.int8_linear import quantize_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [333, 330, 300, 136])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_products_into_a_part(n, dtype):
    rows, d, lib, code = 150, 264, _lib.lib(), _lib.DTYPE_CODE[dtype]
    g = torch.Generator(device="cuda").manual_seed(0)
    x, w = (torch.randint(-3, 4, shape, device="cuda", generator=g).to(dtype) for shape in ((rows, d), (n, d)))
    stream = _lib.stream_ptr(x.device)
    out, back = torch.full((160, 400), 7.0, device="cuda", dtype=dtype), torch.full((160, 400), 7.0, device="cuda", dtype=dtype)
    _lib.check(lib.th_linear_fwd(x.data_ptr(), d, w.data_ptr(), d, None, out.data_ptr(), 400, rows, d, n, code, stream), "th_linear_fwd")
    want = (x.double() @ w.double().t()).to(dtype)  # whole numbers: exact
    assert torch.equal(out[:rows, :n], want) and bool((out[rows:] == 7).all()) and bool((out[:, n:] == 7).all())
    gy = torch.zeros(rows, 336, device="cuda", dtype=dtype)
    gy[:, :n] = torch.randint(-3, 4, (rows, n), device="cuda", generator=g)
    _lib.check(lib.th_linear_bwd_input(gy.data_ptr(), 336, w.data_ptr(), d, back.data_ptr(), 400, rows, d, n, code, stream), "th_linear_bwd_input")
    assert torch.equal(back[:rows, :d], (gy[:, :n].double() @ w.double()).to(dtype)) and bool((back[:, d:] == 7).all()) and bool((back[rows:] == 7).all())
    x8, w8 = quantize_rows(x.float()), quantize_rows(w.float())
    out.fill_(7.0)
    _lib.check(
        lib.th_int8_linear(x8.q.data_ptr(), x8.q.stride(0), x8.scale.data_ptr(), w8.q.data_ptr(), w8.q.stride(0), w8.scale.data_ptr(), None, out.data_ptr(), 400,
                           rows, d, n, code, stream),
        "th_int8_linear",
    )  # fmt: skip
    assert bool((out[rows:] == 7).all()) and bool((out[:, n:] == 7).all())
