"""The serving example: page plans, appends, packed prefill and shared-prefix decode as one loop, its last
step against the paged decode of the same cache. Both round their output to bf16 and one of them its
weights too: for outputs of at most 4 (values are projections of N(0, 1) rows) that is within 2e-2."""
import gc
import importlib.util
from pathlib import Path

import pytest

PATH = Path(__file__).resolve().parents[1] / "examples" / "serve_shared_prefix.py"


@pytest.fixture(autouse=True, scope="module")
def _no_garbage():
    """Tensors that cycles keep (exceptions and their frames, modules) go with the module that made them, not
    in the middle of a later test that counts allocated bytes."""
    yield
    gc.collect()


def example():
    spec = importlib.util.spec_from_file_location("serve_shared_prefix", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def test_the_example_imports_without_a_gpu():
    assert callable(example().serve)


@pytest.mark.gpu
@pytest.mark.parametrize("options", [
    dict(requests=8, prefix=512, prompt=100, steps=6),
    dict(requests=1, prefix=64, prompt=5, steps=2, hq=3, hkv=1, d=64, page_size=24),
    dict(requests=33, prefix=2304, prompt=700, steps=3, hq=32, hkv=8, softcap=30.0),
])
def test_serving_loop(options):
    assert example().serve(**options) <= 2e-2
