"""The operators run as they are used together: a layer's attention (prompt, then decode steps over the cache it has written), whole layers
with experts, and a decode step from hidden states to sampled tokens, eager and as a captured graph.

Tolerances of the attention as in test_kv_attention.py; the projections around it are compared bit for bit with the same kernels
called by themselves."""
import math
import os

import pytest
import torch

import test_kv_attention as A

gpu = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module", params=[True, False], ids=["tcgen05", "mma"])
def lctx(pkg, request):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = pkg.Ctx(0, tcgen05=request.param, pdl=os.environ.get("DSUF_TEST_PDL", "0") == "1")
    yield c
    c.close()


def dense(pkg, ctx, mode, n, k, seed):
    import importlib
    synth = importlib.import_module(pkg.__name__ + ".synth")
    tiles, sds = synth.fp8_dense(torch, mode == pkg.MODE_MX, n, k, 1 / math.sqrt(k), seed, ctx.device)
    return pkg.Weight(ctx, pkg.FMT_FP8, mode, n, k, 1, False, tiles, sds)


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def check_rows(layer, pkg, ctx, rows, want, size):
    A.within(layer.o[:rows], want, size, terms=2 ** -8 + 2 ** -12)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("mode", [0, 1])
def test_attention_layer(pkg, lctx, fp8, mode):
    """Three prompts, then decode steps: the layer's attention against the 64-bit form on the q/k/v rows that its projection gives."""
    ctx, d, hq, hkv, page = lctx, 128, 4, 2, 16
    hidden, lens = 512, [37, 1, 16]
    wqkv, wo = dense(pkg, ctx, mode, (hq + 2 * hkv) * d, hidden, 1), dense(pkg, ctx, mode, hidden, hq * d, 2)
    g = A.gen(4)
    scale = torch.full((hkv,), 0.02, device=DEV)
    cache = pkg.KvCache.empty(ctx, 14, page, hkv, d, fp8, *((scale, scale) if fp8 else ()))
    cos, sin = A.tables(64, d)
    layer = pkg.AttnLayer(ctx, wqkv, wo, cache, hq, 60, rope=(cos, sin, 0))
    t = sum(lens) + 3                                       # three padded rows
    x = A.bf16(g, t, hidden)
    table = torch.randperm(14, generator=g, device=DEV).int()[:12].reshape(3, 4).contiguous()
    pos = i32(*[p for n in lens for p in range(n)], -1, -1, -1)
    seq = i32(*[i for i, n in enumerate(lens) for _ in range(n)], -1, -1, -1)
    cu = i32(0, 37, 38, 54)
    out = torch.empty(t, hidden, dtype=torch.bfloat16, device=DEV)
    layer.prompt(x, pos, seq, cu, table, out)
    # the projection by itself, its rows rotated in 64 bits
    xq, xs = pkg.act_quant(ctx, mode, x)
    rows = pkg.project(ctx, wqkv, xq, xs, torch.empty(t, wqkv.n, dtype=torch.bfloat16, device=DEV))
    n = sum(lens)
    q, k, v = rows[:n].split([hq * d, hkv * d, hkv * d], 1)
    rot = lambda y, at: A.turned64(y.reshape(y.shape[0], -1, d), cos[at.long()], sin[at.long()], 0, False).to(torch.bfloat16).reshape(y.shape[0], -1)   # noqa: E731
    rq, rk = rot(q, pos[:n]), rot(k, pos[:n])
    want, _, size = A.prompt64(rq, rk, v, lens, hq, hkv, d, 0, d ** -0.5)
    # the kernel's rotation rounds to bf16 from fp32 instead of 64 bits: an element may land one bf16 step (2^-7) beside, seldom; the scores
    # move by at most 2^-7 of |q| |k| terms, which the outputs show below 2^-6 of their terms
    A.within(layer.o[:n], want, size, rel=2 ** -8, terms=2 ** -6)
    assert (layer.o[n:t] == 0).all()
    oq, os_ = pkg.act_quant(ctx, mode, layer.o[:t])
    assert torch.equal(out, pkg.project(ctx, wo, oq, os_, torch.empty_like(out)))
    # decode steps; the second step has a padded row
    have = list(lens)
    for step in range(3):
        x1 = A.bf16(g, 3, hidden)
        on = [True, step != 1, True]
        p1 = i32(*[h if o else -1 for h, o in zip(have, on)])
        have = [h + o for h, o in zip(have, on)]
        n1 = i32(*[h if o else 0 for h, o in zip(have, on)])
        out1 = torch.empty(3, hidden, dtype=torch.bfloat16, device=DEV)
        layer.decode(x1, p1, n1, table, out1)
        q1 = layer.qkv[:3, : hq * d]
        want, _, size = A.decode64(cache, q1, table, n1.tolist(), 0, d ** -0.5)
        check_rows(layer, pkg, ctx, 3, want, size)
        oq, os_ = pkg.act_quant(ctx, mode, layer.o[:3])
        assert torch.equal(out1, pkg.project(ctx, wo, oq, os_, torch.empty_like(out1)))
    assert ctx.status().code == 0


def small_stack(pkg, ctx, tokens, **kw):
    import importlib
    stack = importlib.import_module(pkg.__name__ + ".stack")
    cos, sin = A.tables(128, 64)
    cfg = stack.StackConfig(hidden=512, inter=256, n_experts=8, topk=2, layers=2, tokens=tokens, kv_heads=2, head_dim=128, page_size=16, cache_pages=40,
                            rope=(cos, sin, 64), **kw)
    return stack, cfg


@gpu
def test_stack_prompt_then_decode(pkg, lctx):
    """Whole layers: a prompt's last row through the prompt path and the same row as a decode step over the cache of the rows before it
    see the same keys; the attention differs by roundings to bf16 (2^-8), which move one element in sixteen across a border of the e4m3
    activations behind it (2^-4): 2^-6 of the norm for each of six quantizers, 0.04 together."""
    ctx = lctx
    stack, cfg = small_stack(pkg, ctx, 24)
    big = stack.LayerStack(ctx, cfg)
    import copy
    cfg1 = copy.copy(cfg)
    cfg1.tokens = 1
    one = stack.LayerStack(ctx, cfg1, weights_from=big)
    x = A.bf16(A.gen(1), 24, 512)
    table = torch.arange(8, dtype=torch.int32, device=DEV).reshape(1, 8)
    pos, seq = torch.arange(24, dtype=torch.int32, device=DEV), torch.zeros(24, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError):
        big.forward(x)
    for l in range(2):
        one.logits[l].copy_(big.logits[l][23:24])
    y = big.forward(x, step=(pos, seq, i32(0, 24), table)).clone()
    # the decode step writes position 23 again, from the same row of the first layer
    y1 = one.forward(x[23:24].contiguous(), step=(i32(23), i32(24), table))
    torch.cuda.synchronize()
    assert ctx.status().code == 0
    rel = ((y1[0].double() - y[23].double()).norm() / y[23].double().norm()).item()
    assert rel < 0.05, rel


@gpu
@pytest.mark.parametrize("cache_scale", [None, 2.0 ** -7])
def test_decode_step_to_tokens_eager_and_captured(pkg, lctx, cache_scale):
    """Layers -> output head -> sampler, three steps eagerly and as one captured graph replayed with new positions: the same tokens."""
    ctx = lctx
    b, vocab = 5, 1000
    stack, cfg = small_stack(pkg, ctx, b, cache_scale=cache_scale)
    s = stack.LayerStack(ctx, cfg)
    g = A.gen(9)
    head, embed = A.bf16(g, vocab, 512, std=0.2), A.bf16(g, vocab, 512)
    table = torch.arange(b * 8, dtype=torch.int32, device=DEV).reshape(b, 8)
    kw = dict(temperature=torch.full((b,), 0.9, device=DEV), top_k=torch.full((b,), 40, dtype=torch.int32, device=DEV), top_p=torch.full((b,), 0.95, device=DEV))
    tok, pos, lens, u = (torch.zeros(b, dtype=dt, device=DEV) for dt in (torch.int32, torch.int32, torch.int32, torch.float32))
    logits = torch.empty(b, vocab, device=DEV)

    def step():
        y = s.forward(embed[tok.long()], step=(pos, lens, table))
        pkg.lm_head(ctx, head, y, out=logits)
        pkg.sample(ctx, logits, u, ids=tok, **kw)

    def roll(run):
        for a in s.attn:
            a.cache.k.zero_()
            a.cache.v.zero_()
        tok.copy_(torch.arange(b))
        got = []
        for i in range(4):
            pos.fill_(i)
            lens.fill_(i + 1)
            u.copy_(torch.tensor([(0.37 * (i + 1) + 0.13 * j) % 1.0 for j in range(b)]))
            run()
            got.append(tok.clone())
        torch.cuda.synchronize()
        return torch.stack(got).tolist()

    eager = roll(step)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            step()
    torch.cuda.current_stream().wait_stream(side)
    assert roll(graph.replay) == eager
    assert len({t for row in eager for t in row}) > 3 and ctx.status().code == 0
