"""MI355X (gfx950) int8-weight matrix product with telmo's operator surface.

The compute is the HIP library ``lib/libtelmo_hip.so`` behind the C ABI of
``include/telmo_hip.h``; this package mirrors the reference's Python-visible names over it.
"""
from .attention import Attention, PagedCache, Rotary, rotary_frequencies
from .kernels import (Act, E4m3Weights, Epilogue, Kernels, PackedWeights, Precision, TdtDecoder, TelmoError, Token, decode,
                      encode, encode_e4m3, random)
from .pack import Pack
from .sampling import Sampler

__all__ = ["Act", "Attention", "E4m3Weights", "Epilogue", "Kernels", "Pack", "PackedWeights", "PagedCache", "Precision", "Rotary", "Sampler",
           "TdtDecoder", "TelmoError", "Token", "decode", "encode", "encode_e4m3", "random", "rotary_frequencies"]
