"""Calls whose launches would count more than 2^32 work items are refused as arguments, before any device call (no GPU needed)."""
import importlib

import pytest

ARG, BF16 = 1, 1
P = 64  # a pointer that nothing may follow


@pytest.fixture(scope="module")
def h():
    return importlib.import_module("gan-discovery-pso_amd._lib").lib()


@pytest.mark.parametrize("n", [2 ** 30, 2 ** 30 + 65, 2 ** 31 - 1])
def test_code_gradients_of_too_many_rows(h, n):
    """16-bit latents are cut 64 rows a workgroup of 256 threads."""
    ws = h.gdpso_code_logits_grad_workspace_bytes(n, 1, 8)
    assert h.gdpso_code_logits_grad(None, n, 1, 8, P, P, P, BF16, 1.0, P, P, P, ws) == ARG


def test_distill_gradient_of_too_many_long_rows(h):
    """A segment's workgroup has 256 threads, and a row one segment at least."""
    assert h.gdpso_distill_grad(None, 2 ** 24, 2049, 2, P, 2049, 0, P, 0, P, 8, None, 1.0, P, P, P) == ARG


def test_logits_of_too_many_outputs(h):
    """A tile of at most 128 x 128 outputs for every workgroup: 2^31 rows by 2^20 codes."""
    assert h.gdpso_code_logits(None, 2 ** 31 - 1, 300, 2 ** 20, P, P, 0, 1.0, P) == ARG
