"""GPU: the example that runs the rotated append, the shared-prefix attention and the
norm-and-rotation together, with and without sharing the prompt's reads."""
import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "shared_prompt.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("shared_prompt", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


@pytest.mark.parametrize("prompt,seqs,dim", [(600, 3, 128), (512, 8, 64), (777, 24, 128), (1, 6, 32)])
def test_sharing_does_not_change_the_answers(cuda, example, prompt, seqs, dim):
    # Both runs read the same rows; a step's outputs differ by fp16 rounding (about 1e-3), which the next
    # layer's and step's rows carry on: a code of 1 / 7 of the residual's largest flips for some 0.4% of
    # the elements, 2% of a row's rms, in one row of many.
    args = dict(prompt=prompt, seqs=seqs, steps=3, hidden=256, n_heads=8, n_kv_heads=2, head_dim=dim)
    a, b = example.run(**args), example.run(**args, share=False)
    assert torch.isfinite(a["x"]).all()
    assert (a["x"].float() - b["x"].float()).norm() <= 0.02 * b["x"].float().norm()


def test_against_full_precision(cuda, example):
    # Random queries and keys are the worst case of binary scores (a sign row keeps 80% of a vector's
    # norm): the outputs have to be nearer to the exact ones than zeros are.
    r = example.run(prompt=300, seqs=6, steps=2, hidden=256, n_heads=8, n_kv_heads=2, check=True)
    assert len(r["errors"]) == 4 and max(r["errors"]) < 1.0
