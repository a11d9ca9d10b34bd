"""Log probabilities of logits whose difference leaves f32, on the GPU: at a temperature above 1 their
quotient is a finite number again.  Tolerances are those of test_gpu_logprobs.py."""
import numpy as np
import pytest
import torch

from test_gpu_logprobs import case, check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [9, 1500, 5000, 20011, 70001])
@pytest.mark.parametrize("top", [3, 20])
def test_differences_beyond_f32(ctx, io, vocab, top):
    _, t, _ = case(3, 6, vocab, io, "odd")
    t[:] = float("-inf")
    t[:, 1], t[:, vocab // 2], t[:, vocab - 1], t[:, 4], t[:, 2] = 3.2e38, -3.0e38, -1.0e38, 5.0, -3.3e38
    t[3:, 0] = float("inf")  # counts as the largest f32
    temperature = torch.tensor([2.0, 1.0e3, 1.0e36, 2.5, 1.0e30, 5.0e35], device="cuda")
    tokens = torch.tensor([vocab // 2, vocab - 1, 2, 2, vocab // 2, 4], device="cuda")
    got = ctx.token_logprobs(t, tokens, top=top, temperature=temperature)
    assert torch.isfinite(got.logprobs).all() and (got.logprobs < 0).all()
    check(got, t.float().cpu().numpy(), tokens.cpu().numpy(), top, temperature.cpu().numpy())
