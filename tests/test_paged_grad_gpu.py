"""The paged operators have no backward pass: inputs that require a gradient
are refused, and pages written in place count as changed, on the GPU here."""

from __future__ import annotations

import pytest

import paged_grad_cases

pytestmark = pytest.mark.gpu


def test_gradients_are_refused(cuda_device):
    paged_grad_cases.check(cuda_device)
