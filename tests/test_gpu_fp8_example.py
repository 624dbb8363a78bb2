"""The example that trains and serves in 8 bits, at the smallest it is asked for."""
from __future__ import annotations

import importlib.util

import numpy as np
import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example(hip):
    spec = importlib.util.spec_from_file_location("mlp_fp8_small", ROOT / "examples" / "mlp_fp8.py")
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("rows", [1, 3, 8, 40])
def test_answers_as_many_rows_as_there_are(example, rows):
    r = example.main(rows=rows, steps=1)
    assert r["answers"].shape == (min(8, rows), example.LAYERS[-1])
    assert len(r["loss_fp8"]) == 1 and np.isfinite(r["served_error"])


@pytest.mark.parametrize("rows,steps", [(0, 1), (4, 0)])
def test_refuses_no_rows_and_no_steps(example, rows, steps):
    with pytest.raises(ValueError, match="at least one"):
        example.main(rows=rows, steps=steps)
