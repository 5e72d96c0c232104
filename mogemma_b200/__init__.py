"""mogemma_b200: B200 (sm_100a) engine behind the MoGemma Python API.

Public names match the reference package ``mogemma`` (src/py/mogemma/__init__.py)
and are imported lazily.
"""

from importlib import import_module
from typing import TYPE_CHECKING

if TYPE_CHECKING:
    from .config import EmbeddingConfig, GenerationConfig
    from .hub import HubManager
    from .kv8 import KV8Batch as KV8Batch
    from .kv8 import KV8Cache as KV8Cache
    from .model import AsyncGemmaModel, EmbeddingModel, SyncGemmaModel

# KV8Batch and KV8Cache are imported by name: they need torch, which nothing else here does.
__all__ = ["AsyncGemmaModel", "EmbeddingConfig", "EmbeddingModel", "GenerationConfig", "HubManager", "SyncGemmaModel"]

_WHERE = {
    "AsyncGemmaModel": ".model",
    "EmbeddingConfig": ".config",
    "EmbeddingModel": ".model",
    "GenerationConfig": ".config",
    "HubManager": ".hub",
    "KV8Batch": ".kv8",
    "KV8Cache": ".kv8",
    "SyncGemmaModel": ".model",
}


def __getattr__(name: str) -> object:
    where = _WHERE.get(name)
    if where is None:
        msg = f"module 'mogemma_b200' has no attribute '{name}'"
        raise AttributeError(msg)
    value = getattr(import_module(where, __name__), name)
    globals()[name] = value
    return value
