"""vesper_db_b200: B200-native IVF-PQ/OPQ search, exact flat top-k and k-means training
for Vesper, and attention for answering from retrieved passages.

The engine is libvesper_c.so (C++ host code + sm_100a CUDA kernels) exporting the
reference's vesper_ivfpq_* C ABI; this package is its Python mirror.
"""
from ._native import SEARCH_EXACT, SEARCH_FAST, library_path, load  # noqa: F401
from .index import IvfPqIndex, TrainReport, VesperError  # noqa: F401
from .flat import flat_topk, flat_topk_device  # noqa: F401
from .kmeans import KmeansResult, kmeans_cluster, kmeans_elkan, kmeans_fit_device  # noqa: F401

_ATTENTION = ("PageTables", "page_tables", "norm_rotate", "prompt_attention", "shared_prefix_attention")


def __getattr__(name):
    if name in _ATTENTION:  # the attention operators take torch tensors: torch is imported on first use
        try:
            from . import attention
        except (ImportError, RuntimeError) as e:  # without torch or the extension they are not there, and the rest is
            raise AttributeError(f"module {__name__!r} has no {name!r} here: {e}") from e
        globals().update({n: getattr(attention, n) for n in _ATTENTION})
        return globals()[name]
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")


def __dir__():
    return sorted({*globals(), *_ATTENTION})


# What a star import brings; the attention operators, which need torch, come by name.
__all__ = ["IvfPqIndex", "TrainReport", "VesperError", "SEARCH_FAST", "SEARCH_EXACT", "load",
           "library_path", "KmeansResult", "kmeans_cluster", "kmeans_elkan", "kmeans_fit_device",
           "flat_topk", "flat_topk_device"]
