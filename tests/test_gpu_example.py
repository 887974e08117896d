"""The serving example runs the operators together: prompts, samples, graph-captured steps, a compacted cache."""
import importlib.util

import pytest

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("options", [["--steps", "40"], ["--steps", "9", "--window", "0", "--layers", "1"],
                                     ["--samples", "1", "--window", "7", "--sinks", "0", "--steps", "20"]])
def test_serving_example(options, cuda_device):
    """Logits of single tokens against those of whole prompts: both round activations to f16 at the same places, and
    differ by the rounding of other sums (2^-11 a value, through a few layers)."""
    spec = importlib.util.spec_from_file_location("serve", ROOT / "examples" / "serve.py")
    serve = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(serve)
    assert serve.main(options) < 1e-2


def test_serving_example_of_one_step(cuda_device):
    """The first step runs outside the graph: with no other there is nothing to time."""
    spec = importlib.util.spec_from_file_location("serve", ROOT / "examples" / "serve.py")
    serve = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(serve)
    assert serve.main(["--steps", "1"]) < 1e-2
    with pytest.raises(SystemExit):
        serve.main(["--steps", "0"])
