from . import bmm, fused, paged, paged_s4, quantization  # noqa: F401
