"""The serving loop on the paged 4-bit cache (examples/paged_decode.py)."""

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PATH = Path(__file__).resolve().parents[1] / "examples" / "paged_decode.py"


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("kw", [
    dict(layers=2, steps=6), dict(layers=1, steps=9, hq=14, hk=2, d=64, page_size=16, prompts=(1, 16, 90), count=3,
                                  sparse_from=50)])
def test_serving_loop(example, kw):
    # a bf16 output: half an ulp of 2^-8, and weights rounded twice at 2^-11
    assert 0 < example.run(**kw) <= 2.0 ** -8
