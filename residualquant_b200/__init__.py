"""B200-native (sm_100a) packed-KV kernels: the KV-write quantizer and the packed paged decode attention of
ResidualQuant-style KV-cache compression for looped Transformers, behind the reference's operator API.

    from residualquant_b200 import _cuda            # attention(...), quantize(...): reference signatures
    from residualquant_b200.rotation import register_rotation
    from residualquant_b200.block_cache import BlockCache   # 8-bit cache of owners that are not residual-coded
"""

__version__ = "0.1.0"
