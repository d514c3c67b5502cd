"""cqgdn - MI355X (gfx950) gated delta-rule backend, selected as ``gdn_backend: hip``.

``cqgdn.gated_delta_net`` mirrors the reference's ``ops/gated_delta_net.py``; the
kernels live in ``libcqgdn.so`` (C ABI: include/cqgdn.h).  ``cqgdn.rotary``, ``cqgdn.attention`` and
``cqgdn.kvcache`` hold the operators of the attention layers beside the GDN layers: rotary positions, attention over
packed documents with its gradient, pages, the 4-bit and 16-bit caches and the attention over them.
"""

from . import attention, gated_delta_net, kvcache, rotary
from .gated_delta_net import delta, initialize, prefill, provenance, recurrent

__all__ = ["attention", "gated_delta_net", "kvcache", "rotary", "delta", "initialize", "prefill", "provenance", "recurrent"]
