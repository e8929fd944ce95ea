from .kernel import Int8Rows, dequantize_rows, int8_linear, quantize_rows
from .module import Int8Linear


__all__ = ["Int8Rows", "quantize_rows", "dequantize_rows", "int8_linear", "Int8Linear"]
