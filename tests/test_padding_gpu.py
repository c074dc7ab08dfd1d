"""What a batched step makes of rows that only pad the batch and of rows with nothing to draw: no memory that is not the step's own is
read or handed out."""
import numpy as np
import pytest
import torch

from amd_c_b200 import kernels as K
from amd_c_b200 import synth
from amd_c_b200._lib import MAT_F32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cols", [256, 96])
@pytest.mark.parametrize("kind", ["f32", "q4", "q8"])
def test_embed_tokens_that_are_no_rows(cuda, kind, cols):
    """A matrix that is the first half of a larger one: tokens behind its last row give zeros, not the rows that lie there; then the token of
    a row with nothing to draw."""
    rng = np.random.default_rng(cols)
    if kind == "f32":
        whole = K.Mat(MAT_F32, 40, cols, torch.from_numpy(rng.standard_normal((40, cols)).astype(np.float32)).to(cuda))
    else:
        ggml = {"q4": synth.GGML_Q4_0, "q8": synth.GGML_Q8_0}[kind]
        whole = K.Mat.from_gguf(ggml, torch.from_numpy(synth.make_gguf_bytes(ggml, rng, 40, cols)).to(cuda), 40, cols)
    half = K.Mat(whole.kind, 20, cols, whole.data)
    t = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)  # noqa: E731
    rows = K.embed(whole, t(range(40)))
    assert (rows != 0).any(1).all()
    got = K.embed(half, t([19, 20, 0, 39, 5, 21]))
    assert torch.equal(got[[0, 2, 4]], rows[[19, 0, 5]]) and (got[[1, 3, 5]] == 0).all()
    got = K.embed(half, t([-1, 7, -2, 0x7FFFFFFF, 40]))
    assert torch.equal(got[1], rows[7]) and (got[[0, 2, 3, 4]] == 0).all()


def test_tokens_drawn_from_nothing(cuda):
    """Rows of logits without a finite one: their token is -1 (looked at on the host before anything reads it), its embedding zeros."""
    logits = torch.randn(5, 300, device=cuda)
    logits[1], logits[3] = float("nan"), float("-inf")
    idx, prob = K.sample(logits, torch.rand(5, device=cuda), temp=torch.tensor([1.0, 1.0, 0.0, 0.0, 1.0], device=cuda))
    tokens = idx.tolist()
    assert tokens[1] == tokens[3] == -1 and all(0 <= tokens[r] < 300 for r in (0, 2, 4)) and prob.tolist()[1] == prob.tolist()[3] == 0.0
    w = torch.randn(300, 64, device=cuda)
    x = K.embed(K.Mat(MAT_F32, 300, 64, w), idx)
    assert (x[[1, 3]] == 0).all() and torch.equal(x[[0, 2, 4]], w[idx[[0, 2, 4]].long()])
