"""Attention of prompts where scores or values are no finite numbers, on the GPU, against the formula
in 64 bits row by row.  A row that sees a key is never taken for one that sees nothing: scores of NaN
make it NaN, and so do scores of -inf alone, whose log-sum-exp is -inf."""
import numpy as np
import pytest
import torch

from test_gpu_prompt import HALF_STEP, P_STEP, Prompts

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
DIMS = [64, 96, 128, 256]


def expect(p, row, head):
    """(out, lse, tolerance of each) of row (b, i) and head in 64 bits, of the keys it sees and no other; tolerances
    as those of finite inputs (test_gpu_prompt.py), of the finite products."""
    b, i = row
    r, k0 = p.starts[b] + i, p.key_starts[b]
    n = max(0, i + p.nks[b] - p.news[b] + 1)
    if n == 0:
        return np.zeros(p.dim), -INF, np.zeros(p.dim), 0.0
    q = p.q[r, head].double().cpu().numpy()
    k, v = (x[k0:k0 + n, head // p.group].double().cpu().numpy() for x in (p.k, p.v))
    with np.errstate(all="ignore"):
        s = (q * k).sum(-1) * p.dim**-0.5
        ds = 2.0**-24 * (p.dim + 16) * p.dim**-0.5 * np.nan_to_num(np.abs(q * k), nan=0, posinf=0).sum(-1).max()
        sums = 2.0**-24 * (32 + n / 4)
        m = s.max()
        if m == -INF:
            return np.full(p.dim, NAN), -INF, np.zeros(p.dim), 0.0
        e = np.exp(s - m)
        w, z = e / e.sum(), m + np.log(e.sum())
        o = (w[:, None] * v).sum(0)
        tol = (2 * ds + P_STEP[p.io] + sums) * (w[:, None] * np.nan_to_num(np.abs(v), nan=0, posinf=0)).sum(0)
        return o, z, tol + HALF_STEP[p.io] * np.abs(o), ds + sums + 2.0**-23 * (abs(z) + 1)


def rows_of(p):
    return [(b, i, h) for b, n in enumerate(p.news) for i in range(n) for h in range(p.q.shape[1])]


def check(p, got):
    """Where the formula gives no finite number the same, elsewhere within the tolerance."""
    out, lse = got[0].double().cpu().numpy(), got[1].double().cpu().numpy()
    for b, i, h in rows_of(p):
        o, z, tol, ltol = expect(p, (b, i), h)
        y, x, finite, what = out[p.starts[b] + i, h], lse[p.starts[b] + i, h], np.isfinite(o), (p.io, p.dim, b, i, h)
        assert np.array_equal(y[~finite], o[~finite], equal_nan=True), what
        assert (np.abs(y[finite] - o[finite]) <= tol[finite]).all(), what
        assert abs(x - z) <= ltol if np.isfinite(z) else np.array_equal(x, z, equal_nan=True), what


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", [([70, 5], [0, 0]), ([3, 5], [1024, 0])])
def test_a_query_of_nan(ctx, io, dim, news, priors):
    """The row is NaN, log-sum-exp too; no other is.  (Not their bits: rows of a wave move the
    reference of their exponentials together.)"""
    p = Prompts(31, news, priors, 2, 2, dim, io)
    p.q = p.q.clone()
    spoiled = [(0, 1), (news[0] - 1, 3), (int(p.starts[1]), 0)]
    for r, h in spoiled:
        p.q[r, h, 7] = NAN
    got = p.run(ctx)
    check(p, got)
    nan = torch.isnan(got[1])
    assert nan.sum() == len(spoiled) and all(nan[r, h] for r, h in spoiled)
    assert torch.equal(torch.isnan(got[0]), nan[:, :, None].expand_as(got[0]))


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("key", [0, 63, 64, 500, 1023, 1024])
def test_a_key_of_nan(ctx, io, dim, key):
    """One key of NaN, first, last or alone in its part, and all that see it are NaN."""
    p = Prompts(33, [1, 6], [1024, 0], 2, 2, dim, io)
    p.k = p.k.clone()
    p.k[key, 1, 3] = NAN  # of the long sequence
    p.k[1025, 0, 5] = NAN  # the first of the short one: its first row sees nothing else
    got = p.run(ctx)
    check(p, got)
    assert torch.isnan(got[0][0, 2:]).all() and torch.isnan(got[1][0, 2:]).all() and torch.isfinite(got[0][0, :2]).all()
    assert torch.isnan(got[0][1:, :2]).all() and torch.isnan(got[1][1:, :2]).all() and torch.isfinite(got[0][1:, 2:]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("first,last", [(0, 1025), (64, 640), (640, 1025), (0, 700)])
def test_many_keys_of_nan(ctx, io, dim, first, last):
    """All of a part's keys, of all parts' but some, or of all."""
    p = Prompts(35, [1, 2], [1024, 1022], 1, 4, dim, io)
    p.k = p.k.clone()
    p.k[first:last, 0, 9] = NAN
    p.k[1025 + first:1025 + min(last, 1023), 0, 9] = NAN  # its first row does not see the last key
    got = p.run(ctx)
    check(p, got)
    assert torch.isnan(got[0]).all() and torch.isnan(got[1]).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", [([70, 5], [0, 0]), ([2, 5], [1024, 0])])
def test_scores_of_minus_infinity(ctx, dim, news, priors):
    """Keys at -inf have no weight; a row that sees no others is NaN, its log-sum-exp -inf."""
    p = Prompts(37, news, priors, 2, 2, dim, "bf16")
    p.q, p.k = p.q.abs() + 0.125, p.k.clone()
    p.k[:9, 0, 3] = -INF                                             # first keys
    p.k[p.key_starts[1] - 3:p.key_starts[1] - 1, 1, 5] = -INF        # last keys but one
    p.k[p.key_starts[1]:, 0, 5] = -INF                               # all
    p.k[p.key_starts[1], 1, 5] = -INF                                # all that the first row sees
    got = p.run(ctx)
    check(p, got)
    s = int(p.starts[1])
    assert torch.isnan(got[0][s:, :2]).all() and (got[1][s:, :2] == -INF).all() and torch.isnan(got[0][s, 2:]).all()
    assert torch.isfinite(got[0][s + 1:, 2:]).all() and torch.isfinite(got[1][s + 1:, 2:]).all()


@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("prior", [512, 1024, 2048, 4096])
def test_a_part_at_minus_infinity_beside_masked_infinities(ctx, dim, prior):
    """A part whose only key for the row is at -inf, computed by itself for a masked value's sake, while
    the other parts' scores are far below 0."""
    p = Prompts(39, [2], [prior], 1, 1, dim, "bf16")
    p.q, p.k, p.v = torch.full_like(p.q, 2.0), torch.full_like(p.k, -128.0 / dim**0.5), p.v.clone()
    p.k[prior, 0, 0] = -INF
    p.v[prior + 1, 0, 1] = INF
    assert expect(p, (0, 0), 0)[1] < -200
    check(p, p.run(ctx))


SEEN = [([70, 5], [0, 0]), ([1, 5], [1024, 0]), ([40, 1], [3000, 700])]


def small(seed, news, priors, dim, io):
    """Scores so near each other that every weight is a normal f32."""
    p = Prompts(seed, news, priors, 2, 2, dim, io)
    p.q, p.k, p.v = p.q * 0.125, p.k.clone(), p.v.clone()
    return p


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", SEEN)
def test_values_of_infinity(ctx, io, dim, news, priors):
    """Infinite values that all rows see, or the later ones: infinite where they are, and nowhere else; NaN where both
    signs meet."""
    p = small(43, news, priors, dim, io)
    s = int(p.key_starts[1])
    p.v[0, 0, 5], p.v[3, 1, 7], p.v[s, 1, 9] = INF, -INF, INF
    p.v[s - 1, 0, 5], p.v[s - 1, 0, 6] = -INF, INF
    got = p.run(ctx)
    check(p, got)
    assert torch.isnan(got[0][news[0] - 1, :2, 5]).all() and (got[0][news[0] - 1, :2, 6] == INF).all()
    assert (got[0][news[0] - 1, 2:, 7] == -INF).all() and (got[0][news[0]:, 2:, 9] == INF).all()
    assert torch.isfinite(got[1]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", SEEN)
def test_keys_of_infinity(ctx, io, dim, news, priors):
    """A score of -inf has no weight, one of +inf makes the row NaN."""
    p = small(45, news, priors, dim, io)
    p.k[0, 0, 3], p.k[2, 1, 11], p.k[p.key_starts[1], 0, 60] = INF, -INF, -INF
    got = p.run(ctx)
    check(p, got)
    assert torch.isnan(got[0]).any() and torch.isfinite(got[0]).any()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", SEEN)
def test_queries_of_infinity(ctx, io, dim, news, priors):
    """No finite score is left: NaN, and the log-sum-exp -inf where all scores are."""
    p = small(47, news, priors, dim, io)
    p.k[:, 0] = p.k[:, 0].abs() + 0.125
    p.q[0, 0, 3], p.q[0, 1, 3], p.q[-1, 2, 5] = INF, -INF, INF
    got = p.run(ctx)
    check(p, got)
    assert torch.isnan(got[0][0, :2]).all() and torch.isnan(got[1][0, 0]) and got[1][0, 1] == -INF
    assert torch.isfinite(got[0][0, 2:]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 256])
def test_what_sees_nothing_stays_0(ctx, io, dim):
    """Beside keys of NaN rows without keys still give 0 and -inf."""
    p = Prompts(41, [40, 6], [-30, -6], 2, 2, dim, io, key_spare=1)
    p.k = p.k.clone()
    p.k[:, 1, 3] = NAN
    got = p.run(ctx)
    nothing = torch.ones(46, dtype=torch.bool, device="cuda")
    nothing[30:40] = False
    assert (got[0][nothing] == 0).all() and (got[1][nothing] == -INF).all()
    assert torch.isnan(got[0][30:40, 2:]).all() and torch.isnan(got[1][30:40, 2:]).all()
    assert torch.isfinite(got[0][30:40, :2]).all() and torch.isfinite(got[1][30:40, :2]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", [([70, 200], [0, 0]), ([40, 45], [20, 900])])
def test_what_masked_contents_leave(ctx, io, dim, news, priors):
    """The last row's own key and value spoiled, which lie in the tiles of rows before it.  Finite values, however
    large, change no bit of those.  A key of NaN changes none of waves (32 rows of a kv head) that do not hold the
    row that sees it; the others of its wave may move their exponentials' reference elsewhere.  Beside values of
    NaN or infinity rows are summed in another order: within the tolerance, like all of them."""
    p = Prompts(49, news, priors, 2, 2, dim, io)
    clean = p.run(ctx)
    p.check(clean)
    row, key = sum(news) - 1, int(p.key_starts[2]) - 1
    keep_k, keep_v = p.k, p.v
    p.v = keep_v.clone()
    p.v[key] = -3.0e38
    got = p.run(ctx)
    assert torch.equal(got[0][:row], clean[0][:row]) and torch.equal(got[1][:row], clean[1][:row])
    p.k, p.v = keep_k.clone(), keep_v
    p.k[key] = NAN
    got = p.run(ctx)
    alone = int(p.starts[1]) + (2 * news[1] - 1) // 32 * 32 // 2  # the first token of the last wave
    assert alone < row and torch.equal(got[0][:alone], clean[0][:alone]) and torch.equal(got[1][:alone], clean[1][:alone])
    check(p, got)
    for bad in (NAN, INF):
        p.k, p.v = keep_k, keep_v.clone()
        p.v[key, :, 3] = bad
        got = p.run(ctx)
        check(p, got)
        assert torch.equal(got[0][:news[0]], clean[0][:news[0]]) and torch.isfinite(got[0][:row]).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", DIMS)
@pytest.mark.parametrize("news,priors", [([70, 5], [0, 0]), ([1, 5], [1024, 0])])
def test_a_scale_of_0(ctx, io, dim, news, priors):
    """0 times a query that is not finite is NaN; all other rows weigh their keys alike."""
    p = Prompts(51, news, priors, 2, 2, dim, io)
    p.q = p.q.clone()
    for h, x in enumerate((NAN, INF, -INF)):
        p.q[0, h, dim - 1 - h] = x
    got = p.run(ctx, scale=0.0)
    assert torch.isnan(got[0][0, :3]).all() and torch.isnan(got[1][0, :3]).all()
    p.q[0, :3] = 1.0
    out, lse, tol, ltol = p.expect(0.0)
    assert ((got[0].double() - out).abs() <= tol)[1:].all() and ((got[1].double() - lse).abs() <= ltol)[1:].all()
    assert ((got[0].double() - out).abs() <= tol)[0, 3].all()
