"""ash -- torch-ash's Python API on hand-written sm_100a CUDA (B200).

Same public names as the reference package (ash/__init__.py:1-14), and dense layers, norms and
rows in 8 bits that the reference has no native code for.
"""
from .common import DotDict
from .core import ASHEngine, ASHModule
from .embedding import HashEmbedding
from .grid import (
    BoundedSparseDenseGrid,
    SparseDenseGrid,
    UnBoundedSparseDenseGrid,
    UnboundedSparseDenseGrid,
)
from .grid_nns import enumerate_neighbor_coord_offsets
from .grid_query import SparseDenseGridQuery, SparseDenseGridQueryBackward
from .hashmap import HashMap, HashSet
from .mlp import MLP, ResidualMLP, SirenLayer, SirenNet, fused_linear, rms_norm
from .quant import QuantizedRows, dequantize_rows, quantize_rows

__all__ = [
    "ASHEngine", "ASHModule", "BoundedSparseDenseGrid", "DotDict", "HashEmbedding", "HashMap", "HashSet",
    "MLP", "QuantizedRows", "ResidualMLP", "SirenLayer", "SirenNet", "SparseDenseGrid", "SparseDenseGridQuery",
    "SparseDenseGridQueryBackward", "UnBoundedSparseDenseGrid", "UnboundedSparseDenseGrid", "dequantize_rows",
    "enumerate_neighbor_coord_offsets", "fused_linear", "quantize_rows", "rms_norm",
]
