"""cellm_hip_release_graph_scratch without a GPU: a null context is refused."""
from __future__ import annotations

from cellm_amd import _lib


def test_release_of_no_context_is_refused():
    assert _lib.load().cellm_hip_release_graph_scratch(None) == _lib.ERR_INVALID_ARG
    assert "null context" in _lib.last_error()
