"""Refusals of the operators around attention that larger numbers reach."""

import pytest

from .test_decoder_cpu import APPEND, ROTATE, refused


@pytest.mark.parametrize("pairs", [33, 1 << 31, (1 << 62) - 1, 1 << 62, (1 << 62) + 40, (1 << 63) - 1])
def test_more_frequencies_than_pairs(pairs):
    """Twice the number may not fit 64 bits."""
    refused(ROTATE, "ftb_rotate_heads", pairs=pairs)
    refused(APPEND, "ftb_append_heads", pairs=pairs)
