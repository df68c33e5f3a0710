from .linear import sparse_low_precision_linear
from .attention import delta_attention
