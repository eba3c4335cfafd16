"""The paged operators have no backward pass: inputs that require a gradient
are refused, on the CPU here."""

from __future__ import annotations

import paged_grad_cases


def test_gradients_are_refused():
    paged_grad_cases.check("cpu")
