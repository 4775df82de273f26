"""How a cache that keeps every position is held to a fixed size."""
from __future__ import annotations

from dataclasses import dataclass

from ..constants import PAGE


@dataclass(frozen=True)
class CacheEviction:
    """A sequence whose layers without a window hold more than `keep + slack` entries after a step is
    cut down to `keep`: per layer and KV head the entries of the first `sinks` positions stay, those
    of the last `recent` positions, and of the others the ones that attention gave the most
    weight, summed over all queries so far and the heads of the KV head's group.  Positions go on
    counting: an entry keeps the rotation of its own position, and queries see what is stored.

    `slack`: how many entries may come on top before the next cut (a cut costs the same for one
    entry as for many)."""
    keep: int
    recent: int
    sinks: int = 4
    slack: int = PAGE

    def __post_init__(self):
        for name, least in (("keep", 1), ("recent", 0), ("sinks", 0), ("slack", 0)):
            value = getattr(self, name)
            if isinstance(value, bool) or not isinstance(value, int) or value < least:
                raise ValueError(f"{name} must be an integer of at least {least}, got {value!r}")
        if self.sinks + self.recent > self.keep:
            raise ValueError(f"keep {self.keep} does not hold the {self.sinks} first and {self.recent} last positions")
