from . import bmm, fused, paged, quantization  # noqa: F401
