"""B200-native drop-in for the GPU engine of sh1ng/arboretum (hist method)."""
from .core import (ArboretumClassifier, ArboretumError, ArboretumRegression, DMatrix, Garden,
                   build_histogram, lib, load, release_cached_memory, shared_atomic_peak,
                   train)

__all__ = ["ArboretumClassifier", "ArboretumError", "ArboretumRegression", "DMatrix", "Garden",
           "build_histogram", "lib", "load", "release_cached_memory", "shared_atomic_peak", "train",
           "embedding", "embedding_grad", "token_order", "TokenOrder", "AdamW"]

# the operators on torch tensors: torch is imported when one of them is first asked for
_OPERATORS = {"embedding": "lookup", "embedding_grad": "lookup", "token_order": "lookup", "TokenOrder": "lookup",
              "AdamW": "adamw"}


def __getattr__(name):
    if name not in _OPERATORS:
        raise AttributeError("module %r has no attribute %r" % (__name__, name))
    import importlib
    value = getattr(importlib.import_module("." + _OPERATORS[name], __name__), name)
    globals()[name] = value
    return value
