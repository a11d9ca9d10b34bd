"""The speculative decoding example: drafts change the number of rounds, not the tokens."""
import importlib.util
import os

import pytest
import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("speculative_decode", os.path.join(ROOT, "examples", "speculative_decode.py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_greedy_drafts_emit_the_same_tokens(ctx, example):
    """Token for token, up to where the plain run's two best logits are as close as the linears'
    rounding (their kernels differ with the number of rows; 2^-10 of the sums) can move them."""
    model = example.Model(ctx)
    prompts = [[5, 99, 1203, 7, 42], [17, 1999, 3], [11]]
    plain, rounds, logits = example.generate(model, prompts, 40, 0)
    assert rounds == 40
    for depth in (1, 4):
        spec, fewer, _ = example.generate(model, prompts, 40, depth)
        assert fewer < rounds
        for s, (a, b) in enumerate(zip(plain, spec)):
            differs = next((i for i in range(40) if a[i] != b[i]), None)
            if differs is not None:
                row = logits[differs][s]
                assert float(row[a[differs]] - row[b[differs]]) <= 2 ** -6 * float(row.std()), (depth, s, differs)


def test_sampled_runs_are_reproducible(ctx, example):
    model = example.Model(ctx)
    runs = [example.generate(model, [[1, 2, 3], [9]], 24, 3, temperature=0.8, seed=4)[0] for _ in range(2)]
    assert runs[0] == runs[1]
    other = example.generate(model, [[1, 2, 3], [9]], 24, 3, temperature=0.8, seed=5)[0]
    assert other != runs[0]
    torch.cuda.synchronize()
