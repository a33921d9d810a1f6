"""Sizes and settings that the readout operators cannot hold are refused before they touch a GPU."""

from __future__ import annotations

import pytest

from test_readout_boundary import norm, refused


@pytest.mark.parametrize("eps", [1e-50, 1e-46, 7e-46])
def test_norm_refuses_an_eps_that_is_zero_in_float32(eps):
    refused(norm(eps=eps), "eps")
