"""MI355X-native tree-search hot path: device-resident forest, batched PUCT selection with
virtual loss, value backup and leaf gather behind a C ABI (include/omk_forest.h), and what lies
between the search and its network: priors, policy losses and AdamW (include/omk_learn.h)."""
from .forest import Forest, Batch, TranspositionTable, SelectParams, OmkError, library_path, load_library, compact_legal  # noqa: F401
from .learn import Learner, AdamW, pack_legal, legal_of_moves  # noqa: F401

__all__ = ["Learner", "AdamW", "pack_legal", "legal_of_moves", "Forest", "Batch", "TranspositionTable", "SelectParams", "OmkError", "library_path", "load_library", "compact_legal"]
