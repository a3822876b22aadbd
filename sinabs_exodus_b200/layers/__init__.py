"""The EXODUS layers: ``LIF`` and the variants derived from it; the layers on the sequence operators."""
from .lif import LIF
from .sequence import GroupNorm, SelectiveLeak
from .variants import IAF, ExpLeak, ExpLeakSqueeze, IAFSqueeze, LIFSqueeze

__all__ = ["LIF", "LIFSqueeze", "IAF", "IAFSqueeze", "ExpLeak", "ExpLeakSqueeze", "GroupNorm", "SelectiveLeak"]
