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


@pytest.mark.parametrize("io", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [9, 1500, 5000, 20011, 70001])
@pytest.mark.parametrize("warm", [False, True])
def test_rows_that_are_nearly_certain(ctx, io, vocab, warm):
    """A token with almost all of the probability: its logarithm and the entropy are small, and right to their own size.
    With r = S - 1 = sum of e^t over the others, r is off by its own 52 roundings and 4 |t| each, log1p by two of
    its result, U / S as in test_gpu_logprobs.py."""
    rng, t, _ = case(5, 12, vocab, io, "odd", spread=1.0)
    best = rng.integers(0, vocab, 12)
    gap = torch.tensor([3, 5, 8, 11, 14, 17, 20, 25, 30, 45, 60, 80], device="cuda") + float(np.log(vocab))
    t[torch.arange(12), torch.from_numpy(best)] = (torch.tensor([0.0, -40.0, 37.5] * 4, device="cuda") + gap).to(t.dtype)
    t[::3, :] = torch.where(t[::3] == t[::3].amax(1, keepdim=True), t[::3], (t[::3].float() - 2.0).to(t.dtype))
    t[1::3] = torch.where(t[1::3] == t[1::3, torch.from_numpy(best[1::3])].diagonal()[:, None], t[1::3], (t[1::3].float() - 40.0).to(t.dtype))
    t[2::3] = torch.where(t[2::3] == t[2::3, torch.from_numpy(best[2::3])].diagonal()[:, None], t[2::3], (t[2::3].float() + 37.5).to(t.dtype))
    t[4, : vocab // 2] = float("-inf")
    t[4, best[4]] = gap[4].to(t.dtype) - 40.0
    temperature = torch.linspace(0.6, 1.3, 12, device="cuda") if warm else None
    x = t.double().cpu().numpy()
    got = ctx.token_logprobs(t, torch.from_numpy(best).cuda(), top=2, temperature=temperature)
    lp, en, tl = (y.double().cpu().numpy() for y in (got.logprobs, got.entropy, got.top_logprobs))
    small = 0
    for r in range(12):
        temp = 1.0 if temperature is None else float(temperature[r])
        m = x[r].max()
        assert x[r].argmax() == best[r] and (x[r] == m).sum() == 1
        q = (np.delete(x[r], best[r]) - m) / temp
        e, q = np.exp(q), np.where(q > -np.inf, q, 0.0)
        s = e.sum()
        a1, a2, second = (e * -q).sum() / (1 + s), (e * q * q).sum() / (1 + s), q[e > 0].max() if (e > 0).any() else -np.inf
        tol = 2.0**-24 * (52 * s / (1 + s) + 4 * a1 + 3 * np.log1p(s)) + 2.0**-125 * vocab
        assert abs(lp[r] + np.log1p(s)) <= tol and lp[r] == tl[r, 0], (r, lp[r], -np.log1p(s), tol)
        h = np.log1p(s) + a1
        assert abs(en[r] - h) <= tol + 2.0**-24 * (110 * a1 + 4 * a2 + 6 * a1) + 2.0**-118 * vocab, (r, en[r], h)
        assert abs(tl[r, 1] - (second - np.log1p(s))) <= tol + 2.0**-24 * 6 * abs(second)
        small += s < 1e-5
    assert small >= 4 and (lp < 0).sum() >= 8
