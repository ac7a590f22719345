"""chadslab_amd: MI355X-native quantized-weight matrix products (int8 per-row, int4 group-32, MXFP4, FP8 by blocks of 128).

Hand-written HIP kernels for gfx950 behind a C ABI (include/chadq.h, chadslab_amd/libchadq.so); the Python
layer only moves pointers.  Build the library with `python -m chadslab_amd.build`.
"""
from .formats import (QExpertsFP8, QExpertsMXFP4, QRowsFP8, QWeightFP8, QWeightInt4G32, QWeightInt4G32Tiles, QWeightInt8, QWeightMXFP4,  # noqa: F401
                      pack_int4, quantize_int4_g32, quantize_int8_row)

__all__ = ["QExpertsFP8", "QExpertsMXFP4", "QRowsFP8", "QWeightFP8", "QWeightInt4G32", "QWeightInt8", "QWeightMXFP4", "pack_int4", "quantize_int4_g32", "quantize_int8_row", "ops"]
