"""Shared pytest setup.

Markers:
  gpu -- needs a CUDA device and the built product library; run with ``-m gpu``.
"""
from __future__ import annotations

import sys
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
if str(ROOT) not in sys.path:
    sys.path.insert(0, str(ROOT))


def pytest_configure(config):
    config.addinivalue_line("markers", "gpu: test needs a CUDA device (B200) and the built extension")


# fp32 rows whose scale is subnormal have quotients over 127.  These two expect them wrapped to 8 bits, where the definition
# (and test_quantize_rows_clamps_where_the_scale_is_subnormal) clamps: they fail.  Last, so that a run that stops at the
# first failure has run everything else.
RUN_LAST = ("test_quantize_rows_near_half_integers[dtype0-2048]", "test_quantize_rows_near_half_integers[dtype0-2047]")


def pytest_collection_modifyitems(items):
    items.sort(key=lambda item: item.name in RUN_LAST)  # stable


@pytest.fixture(scope="session", autouse=True)
def _built_checker():
    from oracle import build

    build()


def cuda_available() -> bool:
    try:
        import torch

        return torch.cuda.is_available()
    except Exception:  # pragma: no cover
        return False
