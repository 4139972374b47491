"""Keys and values on the device as e4m3 rows (aria_hip_kv of include/aria_hip.h).

``Cache`` owns the codes and the scale bytes of B sequences (or prefixes) and describes them to the
C entry points: ``KVWrite(cache=c.desc, ...)``, ``KVRead(cache=c.desc, ...)``,
``PrefixAttention(prefix=c.desc, own=d.desc, ...)``.
"""
from __future__ import annotations

import numpy as np

from . import KVCache
from .device import DeviceArray


class Cache:
    """Codes [B, heads, slots, D] and bytes [B, heads, slots], uninitialised; slots 0 is an absent cache."""

    def __init__(self, B, heads, slots, D):
        self.B, self.heads, self.slots, self.D = B, heads, slots, D
        self.codes = [DeviceArray((B, heads, slots, D), np.uint8) for _ in range(2)]
        self.scales = [DeviceArray((B, heads, slots), np.uint8) for _ in range(2)]
        self.desc = KVCache(k=self.codes[0].p, v=self.codes[1].p, k_scale=self.scales[0].p, v_scale=self.scales[1].p,
                            batch=heads * slots * D, head=slots * D, token=D, s_batch=heads * slots, s_head=slots, B=B, Hkv=heads,
                            D=D, cap=slots)

    @property
    def nbytes(self):
        return sum(a.nbytes for a in self.codes + self.scales)

    def free(self):
        for a in self.codes + self.scales:
            a.free()
