"""mflux_amd -- MI355X-native group-wise affine quantization and quantized
linears, a drop-in for the MLX operations mflux's diffusion transformers run
through (``mx.quantize`` / ``nn.quantize`` / ``QuantizedLinear`` /
``mx.quantized_matmul``)."""
from . import lora, nn, weights
from .core import (PreparedWeights, dequantize, dequantize_rows, gelu_approx, layer_norm_modulate, prepare_weights, quantize,
                   quantized_matmul,
                   quantized_matmul_epilogue, quantized_matmul_prepared, silu, silu_quantized_matmul)
from .heads import attention, rotary, rotary_tables
from .int8 import int8_dequantize, int8_matmul, int8_quantize, rms_norm, rms_norm_int8

__all__ = ["nn", "lora", "weights", "quantize", "dequantize", "dequantize_rows", "quantized_matmul",
           "quantized_matmul_epilogue", "silu", "gelu_approx", "silu_quantized_matmul", "layer_norm_modulate",
           "prepare_weights", "quantized_matmul_prepared", "PreparedWeights",
           "rotary_tables", "rotary", "attention",
           "rms_norm", "rms_norm_int8", "int8_quantize", "int8_dequantize", "int8_matmul"]
__version__ = "0.1.0"
