"""The example runs: a Gated DeltaNet layer through prefill, fork, decode, verify and compaction."""

import importlib.util
from pathlib import Path

import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("prompt,more", [(150, 6), (5, 16), (64, 1)])
def test_gated_deltanet_example(prompt, more):
    path = Path(__file__).resolve().parent.parent / "examples" / "gated_deltanet.py"
    spec = importlib.util.spec_from_file_location("gated_deltanet_example", path)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.main(prompt=prompt, more=more)
