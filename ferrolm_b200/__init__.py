"""ferrolm_b200: B200 (sm_100a) nearest-neighbour search behind ferrolm's `src/vector` API.

The package is a thin host-side mirror of the reference's Rust interface over the C ABI of
`include/ferrovec.h`; all search code is hand-written CUDA in `csrc/`.  `KvCache` is the same for a language model's keys and
values: rows added (in 16 bits or 8), blocks searched by inner product, attention over them.
"""
from .kv import KvCache
from .vector import (NEIGHBOR, Context, FerrovecError, FlatIndex, Hnsw, HnswParams, IvfPq, IvfPqParams, Metric,
                     datagen, datagen_dev, kmeans_assign, kmeans_train, merge_topk_static, neighbors_from_tensor, normalize, padded,
                     recall)

__all__ = ["NEIGHBOR", "Context", "FerrovecError", "FlatIndex", "Hnsw", "HnswParams", "IvfPq", "IvfPqParams", "KvCache", "Metric",
           "datagen", "datagen_dev", "kmeans_assign", "kmeans_train", "merge_topk_static", "neighbors_from_tensor", "normalize", "padded", "recall"]
