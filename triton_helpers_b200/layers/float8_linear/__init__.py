from .kernel import (
    Float8Blocks,
    dequantize_float8,
    float8_linear,
    float8_training_linear,
    quantize_float8_rows,
    quantize_float8_weight,
)
from .module import Float8Linear, Float8TrainingLinear


__all__ = [
    "Float8Blocks",
    "quantize_float8_rows",
    "quantize_float8_weight",
    "dequantize_float8",
    "float8_linear",
    "float8_training_linear",
    "Float8Linear",
    "Float8TrainingLinear",
]
