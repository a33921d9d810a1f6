"""Sizes and settings that the readout operators cannot hold are refused before they touch a GPU."""

from __future__ import annotations

import pytest

from test_readout_boundary import norm, refused


@pytest.mark.parametrize("eps", [1e-50, 1e-46, 7e-46])
def test_norm_refuses_an_eps_that_is_zero_in_float32(eps):
    refused(norm(eps=eps), "eps")


def test_norm_refuses_columns_past_32_bits():
    """Column numbers are 32-bit in the kernel; only a wide output can ask for so many."""
    for width in ((1 << 30) + 1, (1 << 31) - 1, 1 << 31, (1 << 32) + 5):
        refused(norm(rows=1, width=width, stride=width, scales=None, out_stride=width), "wider than")
