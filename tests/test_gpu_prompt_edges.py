"""Attention of prompts at the edges of what a call may be, on the GPU: broadcast rows, the most heads, layouts of 96 dims,
one workspace for calls after one another, two captured graphs."""
import pytest
import torch

import dyninfer_amd as d
from test_gpu_kvcache import DT, i32, rows
from test_gpu_prompt import HALF_STEP, P_STEP, Prompts

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
@pytest.mark.parametrize("news,priors", [([70, 5], [0, 0]), ([1, 9], [2000, 0])])
def test_broadcast_rows(ctx, io, dim, news, priors):
    """Strides of 0: one key for all tokens, one head of values for all heads, one query for all."""
    p = Prompts(53, news, priors, 3, 2, dim, io)
    p.k = p.k[:1].clone().expand_as(p.k)
    p.v = p.v[:, :1].clone().expand_as(p.v)
    p.check(p.run(ctx))
    p.q = p.q[:1, :1].clone().expand_as(p.q)
    p.check(p.run(ctx, out=torch.empty(p.q.shape, dtype=DT[io], device="cuda")))


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_the_most_heads(ctx, io):
    """65535 query heads on one kv head; one more is refused."""
    gen = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randn(s, device="cuda", generator=gen).to(DT[io])
    q, k, v = new(3, 65535, 64), new(3, 1, 64), new(3, 1, 64)
    batch = d.PromptBatch(i32([0, 2, 3]), 2)
    got = ctx.prompt_attention(q, k, v, batch).double()
    s = torch.einsum("thd,kd->thk", q.double(), k[:, 0].double()) / 8
    see = torch.tensor([[1, 0, 0], [1, 1, 0], [0, 0, 1]], device="cuda").bool()
    w = torch.softmax(s.masked_fill(~see[:, None], float("-inf")), -1)
    ds = 2.0**-24 * 80 * torch.einsum("thd,kd->thk", q.double().abs(), k[:, 0].double().abs()).amax(-1) / 8
    tol = (2 * ds + P_STEP[io] + 2.0**-24 * 33)[..., None] * (w @ v[:, 0].double().abs()) + HALF_STEP[io] * (w @ v[:, 0].double()).abs()
    assert ((got - w @ v[:, 0].double()).abs() <= tol).all()
    with pytest.raises(d.DyninferError):
        ctx.prompt_attention(new(3, 65536, 64), k, v, batch)


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("news,priors", [([1, 64, 65, 200], [0, 0, 0, 0]), ([33, 9], [2500, 700])])
def test_layouts_of_96_dims_have_the_same_bits(ctx, io, news, priors):
    p = Prompts(55, news, priors, 2, 3, 96, io)
    want = p.run(ctx)
    p.check(want)
    tensors = {x: getattr(p, x) for x in "qkv"}
    for how in ("odd", "head_major", "fused"):
        out, _ = rows(p.rng, p.q.shape[0], 6, 96, DT[io], how)
        for x, t in tensors.items():
            y, _ = rows(p.rng, *t.shape, DT[io], how)
            y.copy_(t)
            setattr(p, x, y)
        got = p.run(ctx, out=out)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_one_workspace_in_turn_and_in_two_graphs(ctx, io):
    """What one call leaves in a workspace is nothing to the next, NaN included; graphs that share it are replayed one after
    the other."""
    small, large = Prompts(57, [3, 2], [1500, 900], 1, 2, 128, io), Prompts(58, [40], [3000], 2, 2, 128, io)
    need = [ctx.prompt_attention_workspace_bytes(p.batch(), p.q.shape[0], p.k.shape[0], p.q.shape[1], p.k.shape[1], 128, d._dtype_code(p.q))
            for p in (small, large)]
    assert min(need) > 0
    work = torch.empty(max(need) // 4, dtype=torch.float32, device="cuda").fill_(float("nan"))
    want = [p.run(ctx) for p in (small, large)]
    graphs = []
    for p in (small, large):
        out, lse, batch = torch.empty_like(p.q), torch.empty(p.q.shape[:2], device="cuda"), p.batch()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ctx.prompt_attention(p.q, p.k, p.v, batch, out=out, lse=lse, workspace=work)
        graphs.append((g, out, lse, batch))  # whose tables the graph reads
    for which in (0, 1, 1, 0, 1, 0):
        g, out, lse, _ = graphs[which]
        out.zero_(), lse.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[which][0]) and torch.equal(lse, want[which][1])
        got = (small, large)[1 - which].run(ctx, workspace=work)
        assert torch.equal(got[0], want[1 - which][0]) and torch.equal(got[1], want[1 - which][1])
