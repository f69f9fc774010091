"""The error every binding of libb2g raises on a non-zero status."""
from __future__ import annotations

from . import _lib


class B2GError(RuntimeError):
    def __init__(self, status: int, msg: str):
        super().__init__(f"b2g status {status} ({_lib.STATUS.get(status, '?')}): {msg}")
        self.status = status
