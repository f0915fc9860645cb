"""examples/paged_decode.py: the token-scaled products and the paged cache in a
model's prompt and decode steps, against the same model in plain fp32.

The bound on the logits: rounding n normal values to int8 by their largest (3.3
to 3.7 deviations for these sizes) leaves 0.8% rms, so a product of two such
operands 1.2%; the gated activations' longer tails make that 2%.  Two layers put
four branches of up to 3% (with what they inherit, and the cache's 0.8%) on the
residual, at most 6% together, and the classifier 1.2%; 16-bit activations add
0.4% per rounding.  Twice the sum of these is 15%."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(__file__), "..", "examples", "paged_decode.py")
BOUND = 0.15


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("dtype,dim,heads,kv_heads,page", [
    ("f32", 256, 4, 4, 16), ("f16", 288, 6, 2, 32), ("bf16", 512, 4, 1, 64)])
def test_prompts_and_decode(cuda, example, dtype, dim, heads, kv_heads, page):
    argv = ["--dtype", dtype, "--layers", 2, "--dim", dim, "--hidden", dim + dim // 4, "--heads", heads, "--kv-heads",
            kv_heads, "--vocab", 500, "--seqs", 3, "--prompt", 70, "--page", page, "--steps", 20]
    argv = [str(x) for x in argv]
    first, second = example.main(argv), example.main(argv)
    assert first["error"] < BOUND, first["error"]
    assert (first["context"] - first["context"].new_tensor(first["lengths"])).tolist() == [20, 20, 20]
    assert first["tokens"].shape == (3, 21)
    assert (first["tokens"] == second["tokens"]).all()  # the same tokens every time
