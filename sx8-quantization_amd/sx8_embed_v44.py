"""S-X8 embedding on the kb-major v4.4 layout (graph-capturable, preallocated output).

Interface of scripts/sx8_embed_v44.py (reference): ``ext()`` (an object with
``sx8_embed_v44``) and ``SX8EmbeddingV44``.  The gather kernel is sx8_embed_gather in
libsx8_hip.so; it decodes the selected rows with the canonical R64 recipe, so every
returned row is bit-identical to the same row of decode_tensor_gpu_fast (the
reference's float32 kernel was only within 2e-2).  Ids outside [0, N) leave their
output rows unwritten, as upstream (which skipped ids >= N).
"""
from __future__ import annotations

import torch
import torch.nn as nn

import _sx8lib as _L

DEV = torch.device("cuda")


class _Ext:
    @staticmethod
    def sx8_embed_v44(ids, hdr, levels, basis, scales, K, N, n_cb, out):
        ids_c = ids.reshape(-1).contiguous().to(torch.long)
        T = ids_c.numel()
        if out.numel() < T * int(K) or out.dtype != torch.float16 or not out.is_contiguous():
            raise ValueError("out must be a contiguous float16 tensor of at least (T, K)")
        hb = hdr.shape[1] if hdr.dim() == 2 else 6
        _L.call("sx8_embed_gather", _L.ptr(ids_c), T, _L.ptr(hdr), _L.ptr(levels), int(hb),
                _L.ptr(basis.contiguous()), _L.ptr(scales.contiguous()), int(K), int(N),
                int(n_cb), _L.ptr(out), _L.stream(out.device))
        return out


_ext = None


def ext():
    global _ext
    if _ext is None:
        _L.lib()
        _ext = _Ext()
    return _ext


class SX8EmbeddingV44(nn.Module):
    """Embedding whose table is an S-X8 tensor; output buffer preallocated and reused
    (grow-only), so forward() allocates nothing once warm."""

    def __init__(self, qt, bases_info, hdr_bytes=6):
        super().__init__()
        self.qt = qt
        self.bases_info = bases_info
        self.N = qt["shape"][0]
        self.K = qt["shape"][1]
        self.n_cb = qt["n_cb"]
        self.hdr_bytes = hdr_bytes
        self._t = None
        self._out = None

    def _load(self):
        if self._t is None:
            from sx8_decode1_v3 import make_tensors_v44
            self._t = make_tensors_v44(self.qt, self.bases_info,
                                       hdr_aligned=(self.hdr_bytes == 8))
            self._hdr, self._lvl, self._bas, self._sca = self._t
            self.qt = None
            self.bases_info = None

    def forward(self, ids):
        self._load()
        T = ids.numel()
        if self._out is None or self._out.shape[0] < T:
            self._out = torch.empty(T, self.K, dtype=torch.float16, device=DEV)
        return self.rows(ids, self._out)

    def rows(self, ids, out):
        """The rows of ids, written into the first ones of `out` (at least as many rows, K) fp16: for a caller with a
        buffer of its own, which no later call with more ids replaces."""
        self._load()
        y = _L.py().embed(ids, self._hdr, self._lvl, self._bas, self._sca, self.K, self.N, self.n_cb, out)
        if y is not None:
            return y
        ids_c = ids.reshape(-1).to(torch.long)
        out = out[:ids_c.numel()]
        ext().sx8_embed_v44(ids_c, self._hdr, self._lvl, self._bas, self._sca,
                            self.K, self.N, self.n_cb, out)
        return out.reshape(*ids.shape, self.K)
