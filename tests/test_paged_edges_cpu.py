"""Edges of the paged cache's host side: contexts, size limits of the C entry
points, bookkeeping of pages.  No GPU."""

import pytest
import torch  # noqa: F401


def test_forget_and_sync_without_a_context():
    """A device that no call has used has no context to wait for."""
    from rich_triplet_b200 import paged

    paged._ext.forget(5)
    assert paged._ext.sync(5) is None
    with pytest.raises(TypeError):
        paged._ext.sync()
