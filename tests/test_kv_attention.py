"""Paged cache, decode attention and prompt attention against their definitions in 64 bits.

Tolerances count roundings: a bf16 output is off by at most half a step (2^-8 relative) plus what its inputs' roundings give.
The softmax weights enter the second product rounded to bf16 (2^-8 each, at worst all in one direction), so an output is within
2^-8 of its own magnitude plus 2^-8 of sum_j p_j |v_j|, the sum of its terms' magnitudes; fp32 sums and base-2 exponentials add
less than 2^-12 of that sum (a score s has an absolute error of about d 2^-24 sum |q k| scale, below 2^-14 for these inputs)."""
import math
import os

import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def actx(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = pkg.Ctx(0, pdl=os.environ.get("DSUF_TEST_PDL", "0") == "1")
    yield c
    c.close()


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def bf16(g, *shape, std=1.0):
    return torch.empty(*shape, dtype=torch.bfloat16, device=DEV).normal_(0.0, std, generator=g)


def tables(positions, rot):
    angle = torch.arange(positions, dtype=torch.float64, device=DEV)[:, None] * 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64, device=DEV) * 2 / rot)
    return angle.cos().float(), angle.sin().float()


def turned64(x, cos, sin, off, half):
    """x [t][h][d] with the pairs of columns [off, off + rot) turned, in 64 bits; cos, sin [t][rot / 2]."""
    x = x.double().clone()
    m = cos.shape[1]
    for i in range(m):
        a, b = (off + i, off + i + m) if half else (off + 2 * i, off + 2 * i + 1)
        c, s = cos[:, i].double()[:, None], sin[:, i].double()[:, None]
        u, w = x[..., a].clone(), x[..., b].clone()
        x[..., a], x[..., b] = u * c - w * s, w * c + u * s
    return x


def within(got, want, size, rel=2 ** -8, terms=0.0):
    """|got - want| <= rel |want| + terms size, elementwise; size: the magnitudes of what was added up."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    over = (got - want).abs() - (rel * want.abs() + terms * size + 1e-30)
    assert not torch.isnan(got).any() and over.max().item() <= 0, f"off by {over.max().item()} more than allowed"


def make_cache(pkg, ctx, g, pages, hkv, page, d, fp8, scales=True):
    if fp8:
        k, v = (torch.randn(pages, hkv, page, d, generator=g, device=DEV).mul_(60).clamp_(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for _ in range(2))
        ks, vs = (torch.rand(hkv, generator=g, device=DEV) * 0.02 + 0.01 for _ in range(2)) if scales else (None, None)
        return pkg.KvCache(ctx, k, v, ks, vs)
    return pkg.KvCache(ctx, bf16(g, pages, hkv, page, d), bf16(g, pages, hkv, page, d))


def cache64(cache, scaled=True):
    out = []
    for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)):
        y = x.view(torch.float8_e4m3fn).double() if x.dtype == torch.uint8 else x.double()
        out.append(y * s.double()[None, :, None, None] if scaled and s is not None else y)
    return out


# ------------------------------------------------------------------ append
@gpu
@pytest.mark.parametrize("d,hq,hkv,rot,off,half", [(128, 7, 1, 128, 0, False), (128, 56, 8, 64, 64, False), (64, 3, 3, 64, 0, True), (128, 6, 2, 32, 8, True),
                                                   (64, 0, 5, 16, 40, False), (128, 4, 4, 0, 0, False), (128, 5, 1, 128, 0, True)])
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("t,page", [(1, 16), (37, 32), (700, 128)])
def test_append(pkg, actx, d, hq, hkv, rot, off, half, fp8, t, page):
    g = gen(t + d + hq + rot)
    seqs, pages = 5, max(2, -(-t // 5 // page) + 2)
    cache = make_cache(pkg, actx, g, seqs * pages + 2, hkv, page, d, fp8, scales=rot != 64)
    k_before, v_before = cache.k.clone(), cache.v.clone()
    rows = bf16(g, t, (hq + 2 * hkv) * d + 8)[:, : (hq + 2 * hkv) * d]
    q, k, v = rows.split([hq * d, hkv * d, hkv * d], 1)
    table = torch.randperm(seqs * pages + 2, generator=g, device=DEV)[: seqs * pages].reshape(seqs, pages).int()
    at = torch.arange(t, device=DEV)
    seq, pos = (at % seqs).int(), (at // seqs + page - 3).int()
    pos[at % 11 == 4] = -1                                  # padding tokens
    seq[at % 13 == 5] = -7
    rope = tables(pages * page, rot) if rot else None
    q_out = torch.full((t, hq * d), 7.0, dtype=torch.bfloat16, device=DEV) if hq else None
    pkg.kv_append(actx, cache, k, v, pos, table, seq=seq, rope=(*rope, off) if rot else None, rope_half=half, q=q if hq else None, q_out=q_out)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    live = (pos >= 0) & (seq >= 0)
    p, s = pos[live].long(), seq[live].long()
    cs = [x[p] for x in rope] if rot else [torch.zeros(len(p), 0, device=DEV)] * 2
    page_id = table[s, p // page].long()
    if hq:
        want = turned64(q[live].reshape(-1, hq, d), *cs, off, half)
        size = torch.full_like(want, 0.0)
        # fp32 rotation: three roundings of 2^-24 of the two products' magnitudes
        size += q[live].double().abs().reshape(-1, hq, d).amax(-1, keepdim=True) * 2
        within(q_out[live].reshape(-1, hq, d), want, size, terms=2 ** -22)
        assert (q_out[~live] == 7.0).all()
    for x, before, new, turn, scale in ((cache.k, k_before, k, True, cache.k_scale), (cache.v, v_before, v, False, cache.v_scale)):
        want = new[live].reshape(-1, hkv, d).double()
        size = new[live].double().abs().reshape(-1, hkv, d).amax(-1, keepdim=True).expand_as(want) * 2
        want = turned64(new[live].reshape(-1, hkv, d), *cs, off, half) if turn else want
        got = x[page_id, :, p % page]
        if fp8:
            s = scale.double()[:, None] if scale is not None else 1.0
            got = got.view(torch.float8_e4m3fn)
            # half a step of e4m3: 2^-4 relative, 2^-10 below its normal range; the fp32 value before it is off by 2^-22
            within(got, (want / s).clamp(-448, 448), size / s + 2 ** -10 * 2 ** 22, rel=2 ** -4 * 1.0001, terms=2 ** -22)
        else:
            within(got, want, size, terms=2 ** -22)
        touched = torch.zeros(x.shape[0], page, dtype=torch.bool, device=DEV)
        touched[page_id, p % page] = True
        same = (x.view(torch.uint8) == before.view(torch.uint8)).reshape(x.shape[0], hkv, page, -1).all(-1).all(1)
        assert same[~touched].all()                         # nothing else of the cache is written


@gpu
def test_append_in_place_and_bad_indexes(pkg, actx):
    g = gen(3)
    d, hq, hkv, page = 128, 4, 2, 16
    cache = make_cache(pkg, actx, g, 6, hkv, page, d, False)
    q, k, v = bf16(g, 4, hq * d), bf16(g, 4, hkv * d), bf16(g, 4, hkv * d)
    cos, sin = tables(40, 128)
    table = torch.tensor([[0, 1], [2, 99], [3, -1]], dtype=torch.int32, device=DEV)
    for half in (False, True):
        fresh = pkg.kv_append(actx, cache, k, v, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV), table,
                              seq=torch.tensor([0, 1, 2, 0], dtype=torch.int32, device=DEV), rope=(cos, sin, 0), rope_half=half, q=q)
        again = q.clone()
        pkg.kv_append(actx, cache, k, v, torch.tensor([0, 1, 2, 3], dtype=torch.int32, device=DEV), table,
                      seq=torch.tensor([0, 1, 2, 0], dtype=torch.int32, device=DEV), rope=(cos, sin, 0), rope_half=half, q=again, q_out=again)
        assert torch.equal(fresh, again)
    assert actx.status().code == 0
    before = cache.k.clone()
    # a page beyond the cache, a negative page, a sequence and a position beyond the table: each alone is reported and skipped
    for seq, pos in ((1, 17), (2, 16), (3, 0), (0, 32)):
        pkg.kv_append(actx, cache, k[:1], v[:1], torch.tensor([pos], dtype=torch.int32, device=DEV), table,
                      seq=torch.tensor([seq], dtype=torch.int32, device=DEV), rope=(cos, sin, 0))
        with pytest.raises(pkg.DsufError, match="status 2 from kernel 7"):
            actx.status()
    short = (cos[:10].contiguous(), sin[:10].contiguous(), 0)
    pkg.kv_append(actx, cache, k[:1], v[:1], torch.tensor([12], dtype=torch.int32, device=DEV), table, rope=short)
    with pytest.raises(pkg.DsufError):
        actx.status()
    assert torch.equal(before, cache.k) and actx.status().code == 0


# ------------------------------------------------------------------ decode
def decode64(cache, q, table, lens, window, scale, with_size=False):
    b, hq, d = q.shape[0], q.shape[1] // cache.head_dim, cache.head_dim
    k, v = cache64(cache)
    out = torch.zeros(b, hq, d, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    lse = torch.full((b, hq), -math.inf, dtype=torch.float64, device=DEV)
    g = hq // cache.kv_heads
    for i, n in enumerate(lens):
        lo = max(0, n - window) if window else 0
        if n <= 0:
            continue
        pg = table[i, : -(-n // cache.page_size)].long()
        for h in range(hq):
            kk, vv = (x[pg, h // g].reshape(-1, d)[lo:n] for x in (k, v))
            s = (kk @ q[i].double().reshape(hq, d)[h]) * scale
            lse[i, h] = torch.logsumexp(s, 0)
            p = torch.softmax(s, 0)
            out[i, h], size[i, h] = p @ vv, p @ vv.abs()
    return out.reshape(b, -1), lse, size.reshape(b, -1)


def decode_inputs(pkg, ctx, seed, lens, hq, hkv, d, page, fp8, poison=False):
    g = gen(seed)
    per = [max(1, -(-n // page)) for n in lens]
    cache = make_cache(pkg, ctx, g, sum(per) + 3, hkv, page, d, fp8)
    order = torch.randperm(sum(per) + 3, generator=g, device=DEV).int()
    table = torch.full((len(lens), max(per) + 1), -1, dtype=torch.int32, device=DEV)   # behind a sequence: no page at all
    if poison:   # every slot that no sequence sees holds NaN
        nan = 0x7f if fp8 else 0x7fc0
        seen = torch.zeros(sum(per) + 3, page, dtype=torch.bool, device=DEV)
    e = 0
    for i, n in enumerate(per):
        table[i, :n] = order[e: e + n]
        if poison:
            for j in range(lens[i]):
                seen[order[e + j // page].long(), j % page] = True
        e += n
    if poison:
        for x in (cache.k, cache.v):
            raw = x if fp8 else x.view(torch.int16)
            raw[~seen[:, None, :, None].expand_as(x)] = nan
    q = bf16(g, len(lens), hq * d + 16, std=1.5)[:, : hq * d]
    return cache, q, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (16, 2), (12, 1), (34, 2), (8, 8)])
@pytest.mark.parametrize("lens,page,window", [([1], 16, 0), ([0, 5, 16, 17, 0, 64, 65, 300], 16, 0), ([1000, 1, 129], 32, 128), ([3001], 64, 0),
                                              ([40, 500, 31], 128, 33), ([700, 2], 16, 1)])
def test_decode(pkg, actx, fp8, d, hq, hkv, lens, page, window):
    cache, q, table, n = decode_inputs(pkg, actx, 5 + len(lens) + hq, lens, hq, hkv, d, page, fp8, poison=True)
    out, lse = pkg.attn_decode(actx, cache, q, table, n, window=window, return_lse=True)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    if fp8:   # (the 64-bit form multiplies what no sequence sees by nothing, but must not meet NaN in the pages it reads)
        for x in (cache.k, cache.v):
            x[x == 0x7f] = 0
    else:
        for x in (cache.k, cache.v):
            x.nan_to_num_(0)
    want, wl, size = decode64(cache, q, table, lens, window, d ** -0.5)
    within(out, want, size, terms=2 ** -8 + 2 ** -12)
    live = wl > -math.inf
    assert torch.equal(live, lse > -math.inf)
    assert ((lse.double() - wl)[live].abs() <= 2 ** -12 + 2 ** -22 * wl[live].abs()).all()
    again = pkg.attn_decode(actx, cache, q, table, n, window=window)
    assert torch.equal(out, again)                          # the join's order does not depend on timing


# ------------------------------------------------------------------ prompt
def prompt64(q, k, v, lens, hq, hkv, d, window, scale):
    t = q.shape[0]
    q, k, v = (x.double().reshape(t, -1, d) for x in (q, k, v))
    out = torch.zeros(t, hq, d, dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    lse = torch.zeros(t, hq, dtype=torch.float64, device=DEV)
    b = 0
    for n in lens:
        i = torch.arange(n, device=DEV)
        hidden = i[None, :] > i[:, None]
        if window:
            hidden |= i[None, :] <= i[:, None] - window
        for h in range(hq if n else 0):
            s = (q[b: b + n, h] @ k[b: b + n, h // (hq // hkv)].T * scale).masked_fill(hidden, -math.inf)
            p = torch.softmax(s, 1)
            lse[b: b + n, h] = torch.logsumexp(s, 1)
            out[b: b + n, h] = p @ v[b: b + n, h // (hq // hkv)]
            size[b: b + n, h] = p @ v[b: b + n, h // (hq // hkv)].abs()
        b += n
    return out.reshape(t, -1), lse, size.reshape(t, -1)


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv", [(1, 1), (7, 1), (6, 3), (5, 5), (16, 2)])
@pytest.mark.parametrize("lens,window", [([1], 0), ([128], 0), ([129, 0, 127, 1, 300], 0), ([700], 0), ([1000, 3, 257], 128), ([400, 131], 1), ([900], 333),
                                         ([5] * 70, 0)])
def test_prompt(pkg, actx, d, hq, hkv, lens, window):
    g = gen(sum(lens) + hq + d)
    t = sum(lens) + 9                                       # rows behind the last sequence
    rows = bf16(g, t, (hq + 2 * hkv) * d)
    rows[sum(lens):] = math.nan
    q, k, v = rows.split([hq * d, hkv * d, hkv * d], 1)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    out = torch.full((t, hq * d), 5.0, dtype=torch.bfloat16, device=DEV)
    lse = torch.full((t, hq), 5.0, device=DEV)
    pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window, out=out, lse=lse)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    n = sum(lens)
    assert (out[n:] == 5.0).all() and (lse[n:] == 5.0).all()
    want, wl, size = prompt64(q[:n], k[:n], v[:n], lens, hq, hkv, d, window, d ** -0.5)
    within(out[:n], want, size, terms=2 ** -8 + 2 ** -12)
    assert ((lse[:n].double() - wl).abs() <= 2 ** -12 + 2 ** -22 * wl.abs()).all()
    again = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window)
    assert torch.equal(out[:n], again[:n])


# ------------------------------------------------------------------ strides, streams, workspaces
@gpu
@pytest.mark.parametrize("hq,hkv", [(3, 1), (4, 2), (5, 1)])
@pytest.mark.parametrize("window", [0, 100])
def test_prompt_of_many_sequences(pkg, actx, hq, hkv, window):
    """More sequences than a warp looks at together, of all lengths, so that every level of the deal takes from several groups of 32."""
    d = 64
    lens = [(53 * i * i) % 700 if i % 5 else 0 for i in range(75)]
    g = gen(81 + hq)
    t = sum(lens)
    q, k, v = bf16(g, t, hq * d), bf16(g, t, hkv * d), bf16(g, t, hkv * d)
    cu = torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    out = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    want, _, size = prompt64(q, k, v, lens, hq, hkv, d, window, d ** -0.5)
    within(out.reshape(want.shape), want, size, terms=2 ** -8 + 2 ** -12)


@gpu
@pytest.mark.parametrize("d,window", [(128, 1024), (64, 1000), (128, 127), (64, 129), (128, 255), (64, 32)])
def test_prompt_windows_over_many_tiles(pkg, actx, d, window):
    """Windows that end on, before and behind a tile's border, with scores that differ by far more inside a row than in its first columns."""
    lens, hq, hkv = [2300, 1, 700], 6, 2
    g = gen(71 + window)
    t = sum(lens)
    q, k, v = bf16(g, t, hq * d, std=3.0), bf16(g, t, hkv * d, std=2.0), bf16(g, t, hkv * d)
    cu = torch.tensor([0, 2300, 2301, 3001], dtype=torch.int32, device=DEV)
    out, lse = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window, return_lse=True)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    want, wl, size = prompt64(q, k, v, lens, hq, hkv, d, window, d ** -0.5)
    within(out.reshape(want.shape), want, size, terms=2 ** -8 + 2 ** -12)
    assert ((lse.double() - wl).abs() <= 2 ** -12 + 2 ** -20 * wl.abs()).all()


@gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_interleaved_layers_and_far_pages(pkg, actx, fp8):
    """Pages of two layers interleaved in one allocation (a page stride of its own), and a pool of more than 2^31 elements, so that an offset
    into it passes 32 bits."""
    d, hkv, page, far = 128, 8, 64, 33000                    # 33000 * 8 * 64 * 128 = 2.16e9 elements per layer of k
    dt = torch.uint8 if fp8 else torch.bfloat16
    pool = torch.zeros(far, hkv, page, d, dtype=dt, device=DEV)
    both = torch.zeros(6, 2, hkv, page, d, dtype=dt, device=DEV)
    g = gen(8)
    k, v, q = bf16(g, 3, hkv * d), bf16(g, 3, hkv * d), bf16(g, 3, 2 * hkv * d)
    pos = torch.tensor([0, 63, 64], dtype=torch.int32, device=DEV)
    for cache, table in ((pkg.KvCache(actx, pool, pool.clone()), torch.tensor([[far - 1, far - 7]], dtype=torch.int32, device=DEV)),
                         (pkg.KvCache(actx, both[:, 1], both.clone()[:, 1]), torch.tensor([[5, 2]], dtype=torch.int32, device=DEV))):
        pkg.kv_append(actx, cache, k, v, pos, table, seq=torch.zeros(3, dtype=torch.int32, device=DEV))
        assert (cache.k[table[0, 0].long(), :, 0] != 0).any() and (cache.v[table[0, 1].long(), :, 0] != 0).any()
        out = pkg.attn_decode(actx, cache, q[:1], table, torch.tensor([65], dtype=torch.int32, device=DEV))
        live = table[0].long()
        small = pkg.KvCache(actx, cache.k[live].contiguous(), cache.v[live].contiguous())
        want, _, size = decode64(small, q[:1], torch.tensor([[0, 1]], dtype=torch.int32, device=DEV), [65], 0, d ** -0.5)
        within(out, want, size, terms=2 ** -8 + 2 ** -12)
    assert (both[:, 0] == 0).all() and actx.status().code == 0


@gpu
def test_two_streams_with_workspaces_of_their_own(pkg, actx):
    cache, q, table, n = decode_inputs(pkg, actx, 3, [4000, 77, 1500], 8, 2, 128, 32, False)
    alone = pkg.attn_decode(actx, cache, q, table, n)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [actx.attn_workspace, actx.new_attn_workspace()]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for st, w in zip(streams, spaces):
            with torch.cuda.stream(st):
                got.append(pkg.attn_decode(actx, cache, q, table, n, workspace=w))
    torch.cuda.synchronize()
    assert all(torch.equal(alone, x) for x in got)


@gpu
def test_captured_decode_follows_new_lengths(pkg, actx):
    cache, q, table, n = decode_inputs(pkg, actx, 7, [900, 300, 2000, 31], 6, 2, 64, 16, True)
    out = torch.empty(4, 6 * 64, dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            pkg.attn_decode(actx, cache, q, table, n, out=out)
    torch.cuda.current_stream().wait_stream(side)
    for lens in ([900, 300, 2000, 31], [1, 0, 16, 17], [0, 0, 0, 0], [333, 300, 1, 30]):
        n.copy_(torch.tensor(lens))
        graph.replay()
        assert torch.equal(out, pkg.attn_decode(actx, cache, q, table, n))


@gpu
def test_many_sequences(pkg, actx):
    """More sequences than a warp has lanes, most of them empty or of one token, next to a long one."""
    lens = [0] * 700
    for i in range(0, 700, 7):
        lens[i] = 1 + i % 40
    lens[333], lens[699] = 5000, 3
    cache, q, table, n = decode_inputs(pkg, actx, 11, lens, 3, 1, 64, 16, False)
    out, lse = pkg.attn_decode(actx, cache, q, table, n, return_lse=True)
    want, wl, size = decode64(cache, q, table, lens, 0, 64 ** -0.5)
    within(out, want, size, terms=2 ** -8 + 2 ** -12)
    assert torch.equal(wl > -math.inf, lse > -math.inf)


@gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("d,hq,hkv,window", [(128, 56, 8, 0), (128, 12, 1, 0), (64, 34, 2, 70), (64, 3, 3, 1)])
@pytest.mark.parametrize("most", [1, 17, 65, 256])
def test_many_short_sequences(pkg, actx, fp8, d, hq, hkv, window, most):
    """Enough short contexts for every SM: each of 0 to `most` tokens."""
    lens = [(37 * i) % (most + 1) for i in range(600)]
    cache, q, table, n = decode_inputs(pkg, actx, 21 + most, lens, hq, hkv, d, 16, fp8)
    out, lse = pkg.attn_decode(actx, cache, q, table, n, window=window, return_lse=True)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    want, wl, size = decode64(cache, q, table, lens, window, d ** -0.5)
    within(out, want, size, terms=2 ** -8 + 2 ** -12)
    live = wl > -math.inf
    assert torch.equal(live, lse > -math.inf)
    assert ((lse.double() - wl)[live].abs() <= 2 ** -12 + 2 ** -22 * wl[live].abs()).all()


@gpu
@pytest.mark.parametrize("lens", [[3000, 5], [40] * 400])
def test_decode_in_place_and_over_shared_pages(pkg, actx, lens):
    """out = q, by ranges and by warps, and sequences that all read the first one's pages."""
    cache, q, table, n = decode_inputs(pkg, actx, 51, lens, 16, 2, 128, 16, False)
    want, lse = pkg.attn_decode(actx, cache, q, table, n, return_lse=True)
    mine = q.clone()
    assert pkg.attn_decode(actx, cache, mine, table, n, out=mine) is mine
    assert torch.equal(mine, want)
    first = table[:1].repeat(len(lens), 1)
    n.fill_(lens[0])
    got = pkg.attn_decode(actx, cache, q[:1].repeat(len(lens), 1), first, n)
    torch.cuda.synchronize()
    assert actx.status().code == 0
    want, _, size = decode64(cache, q[:1].repeat(len(lens), 1), first, [lens[0]] * len(lens), 0, 128 ** -0.5)
    within(got, want, size, terms=2 ** -8 + 2 ** -12)


@gpu
def test_a_new_workspace_is_ready_for_another_stream(pkg, actx):
    cache, q, table, n = decode_inputs(pkg, actx, 53, [5000], 8, 1, 128, 16, False)
    want = pkg.attn_decode(actx, cache, q, table, n)
    junk = torch.full((64 << 20,), 255, dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    for _ in range(4):
        for _ in range(20):
            junk.add_(0)                 # keeps the creating stream busy
        w = torch.full_like(actx.attn_workspace, 255)
        del w                            # (its memory is what the new one gets)
        w = actx.new_attn_workspace()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = pkg.attn_decode(actx, cache, q, table, n, workspace=w)
        side.synchronize()
        assert torch.equal(got, want)


@gpu
def test_every_bad_length_is_reported(pkg, actx):
    """One length beyond its table among many short contexts, wherever it stands, is cut to the table and reported."""
    lens = [5] * 600
    cache, q, table, n = decode_inputs(pkg, actx, 31, lens, 7, 1, 64, 16, False)
    want = pkg.attn_decode(actx, cache, q, table, n)
    table = table[:, :1].contiguous()
    for at in (0, 1, 299, 599):
        n[at] = 17
        got = pkg.attn_decode(actx, cache, q, table, n)
        with pytest.raises(pkg.DsufError, match="status 2 from kernel 8"):
            actx.status()
        n[at] = 16
        assert torch.equal(got, pkg.attn_decode(actx, cache, q, table, n)) and actx.status().code == 0
        n[at] = 5
    assert torch.equal(want, pkg.attn_decode(actx, cache, q, table, n))


@gpu
def test_bad_pages_and_lengths_are_reported(pkg, actx):
    cache, q, table, n = decode_inputs(pkg, actx, 12, [100, 40], 4, 2, 128, 16, False)
    good = pkg.attn_decode(actx, cache, q, table, n)
    bad = table.clone()
    bad[0, 2] = cache.n_pages
    out = pkg.attn_decode(actx, cache, q, bad, n)
    with pytest.raises(pkg.DsufError, match="status 2 from kernel 8"):
        actx.status()
    assert torch.equal(out[1], good[1]) and not torch.isnan(out).any()
    pkg.attn_decode(actx, cache, q, table, torch.tensor([100, 10 ** 9], dtype=torch.int32, device=DEV))
    with pytest.raises(pkg.DsufError, match="status 2 from kernel 8"):
        actx.status()
    assert torch.equal(good, pkg.attn_decode(actx, cache, q, table, n)) and actx.status().code == 0


@gpu
def test_large_scores_move_the_reference(pkg, actx):
    """Scores that grow along the context by far more than the reference's slack, in both kernels, and scores of thousands."""
    g = gen(21)
    d, n = 128, 700
    q, k, v = bf16(g, n, 2 * d), bf16(g, n, d), bf16(g, n, d)
    k *= (1.0 + torch.arange(n, device=DEV)[:, None] * 0.2).to(torch.bfloat16)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    for scale in (d ** -0.5, 1.0, 20.0):
        out, lse = pkg.attn_prompt(actx, q, k, v, cu, scale=scale, return_lse=True)
        want, wl, size = prompt64(q, k, v, [n], 2, 1, d, 0, scale)
        # a score of magnitude s carries an fp32 error of up to 128 2^-24 s' (s' the sum of its terms' magnitudes): with s' below 2^17 here that
        # is below 1 at scale 20, so outputs are only compared where the largest weight is beyond doubt
        if scale < 1:
            within(out, want, size, terms=2 ** -8 + 2 ** -6)
        assert not torch.isnan(out).any() and ((lse.double() - wl).abs() <= 2 ** -12 + 2 ** -16 * wl.abs() + 128 * 2.0 ** -24 * scale * 2 ** 17).all()
        cache = pkg.KvCache.empty(actx, 44, 16, 1, d)
        table = torch.arange(44, dtype=torch.int32, device=DEV).reshape(1, 44)
        pkg.kv_append(actx, cache, k, v, torch.arange(n, dtype=torch.int32, device=DEV), table, seq=torch.zeros(n, dtype=torch.int32, device=DEV))
        o1, l1 = pkg.attn_decode(actx, cache, q[-1:], table, torch.tensor([n], dtype=torch.int32, device=DEV), scale=scale, return_lse=True)
        if scale < 1:
            within(o1, want[-1:], size[-1:], terms=2 ** -8 + 2 ** -6)
        assert ((l1.double() - wl[-1:]).abs() <= 2 ** -12 + 2 ** -16 * wl[-1:].abs() + 128 * 2.0 ** -24 * scale * 2 ** 17).all()


@gpu
@pytest.mark.parametrize("score", [-8e31, 8e31, -1e37, 1e37])
def test_scores_near_the_ends_of_fp32(pkg, actx, score):
    """All scores equal and huge: the plain mean of the visible values, with and without a window."""
    g = gen(61)
    d, n = 64, 300
    q = torch.ones(n, 2 * d, dtype=torch.bfloat16, device=DEV)
    k = torch.full((n, d), score / 8, dtype=torch.float32, device=DEV).bfloat16()      # (times 64 columns times the scale 1/8: the score)
    v = bf16(g, n, d)
    cu = torch.tensor([0, n], dtype=torch.int32, device=DEV)
    for window in (0, 50):
        out = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window).double().reshape(n, 2, d)
        for r in (0, 1, 49, 128, 299):
            seen = v.double()[max(0, r + 1 - window) if window else 0: r + 1]
            within(out[r], seen.mean(0).expand(2, d), seen.abs().mean(0).expand(2, d), terms=2 ** -8 + 2 ** -12)
    cache = pkg.KvCache.empty(actx, 20, 16, 1, d)
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    table = torch.arange(19, dtype=torch.int32, device=DEV)[None]
    pkg.kv_append(actx, cache, k, v, pos, table, seq=torch.zeros_like(pos))
    for window in (0, 50):
        seen = v.double()[n - window if window else 0:]
        out = pkg.attn_decode(actx, cache, q[:1], table, pos[-1:] + 1, window=window).double().reshape(2, d)
        within(out, seen.mean(0).expand(2, d), seen.abs().mean(0).expand(2, d), terms=2 ** -8 + 2 ** -12)


@gpu
def test_nan_stays_with_the_rows_that_see_it(pkg, actx):
    g = gen(22)
    d, lens = 64, [200, 60]
    q, k, v = bf16(g, 260, d), bf16(g, 260, d), bf16(g, 260, d)
    cu = torch.tensor([0, 200, 260], dtype=torch.int32, device=DEV)
    clean = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d)
    k2 = k.clone()
    k2[150, 3] = math.nan                                   # seen by rows 150 .. 199
    out = pkg.attn_prompt(actx, q, k2, v, cu, head_dim=d)
    assert torch.equal(out[:150], clean[:150]) and torch.equal(out[200:], clean[200:]) and torch.isnan(out[150:200]).all()
    v2 = v.clone()
    v2[200:] = math.inf                                     # the next sequence's values, in the first one's last tile
    out = pkg.attn_prompt(actx, q, k, v2, cu, head_dim=d)
    assert torch.equal(out[:200], clean[:200])


# ------------------------------------------------------------------ refusals
@gpu
def test_refusals(pkg, actx):
    E, d = pkg.DsufError, 128
    z = lambda *s, dt=torch.bfloat16, dev=DEV: torch.zeros(*s, dtype=dt, device=dev)   # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)   # noqa: E731
    cache = pkg.KvCache.empty(actx, 4, 16, 2, d)
    k, v, q, pos, table = z(3, 2 * d), z(3, 2 * d), z(3, 4 * d), i(3), i(3, 1)
    ok = dict(ctx=actx, cache=cache, k=k, v=v, pos=pos, block_table=table)
    pkg.kv_append(**ok)
    bad_append = [dict(k=k.float()), dict(k=k.cpu()), dict(k=z(3, d)), dict(v=z(2, 2 * d)), dict(pos=pos.long()), dict(pos=i(2)), dict(pos=i(6)[::2]),
                  dict(block_table=i(3)), dict(block_table=i(2, 1)), dict(seq=i(2)), dict(q=z(3, d + 8)), dict(q=z(3, 0)), dict(q=q, q_out=z(3, 2 * d)),
                  dict(k=z(3, 2 * d + 1)[:, 1:]), dict(k=z(3, 2 * d + 4)[:, : 2 * d]), dict(k_out=z(3, d)), dict(rope=(z(8, 4), z(8, 4), 0)),
                  dict(rope=(z(8, 4, dt=torch.float32), z(8, 4, dt=torch.float32), 0)), dict(rope=(z(8, 64, dt=torch.float32), z(8, 32, dt=torch.float32), 0)),
                  dict(rope=(z(8, 64, dt=torch.float32), z(8, 64, dt=torch.float32), 8)), dict(rope=(z(8, 32, dt=torch.float32), z(8, 32, dt=torch.float32), 4)),
                  dict(k=[1, 2]), dict(k=None)]
    for b in bad_append:
        with pytest.raises(E):
            pkg.kv_append(**{**ok, **b})
    okd = dict(ctx=actx, cache=cache, q=q, block_table=table, seq_lens=pos)
    pkg.attn_decode(**okd)
    for b in [dict(q=z(3, 3 * d)), dict(q=z(3, 0)), dict(q=q.half()), dict(q=z(3, 4 * d + 2)[:, : 4 * d]), dict(block_table=i(2, 1)), dict(seq_lens=i(4)), dict(seq_lens=pos.float()),
              dict(out=z(3, 2 * d)), dict(lse=z(3, 3, dt=torch.float32)), dict(lse=z(3, 4)), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan), dict(scale=math.inf),
              dict(window=-1), dict(workspace=z(16, dt=torch.uint8))]:
        with pytest.raises(E):
            pkg.attn_decode(**{**okd, **b})
    cu = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
    okp = dict(ctx=actx, q=q, k=k, v=v, cu_seqlens=cu, head_dim=d)
    pkg.attn_prompt(**okp)
    for b in [dict(head_dim=96), dict(head_dim=32), dict(q=z(3, 3 * d)), dict(k=z(2, 2 * d)), dict(v=z(3, d)), dict(cu_seqlens=cu.long()), dict(cu_seqlens=i(0)), dict(out=z(3, d)),
              dict(lse=z(4, 3, dt=torch.float32)), dict(scale=0.0), dict(scale=math.nan), dict(window=-2), dict(q=z(3, 4 * d + 4)[:, : 4 * d])]:
        with pytest.raises(E):
            pkg.attn_prompt(**{**okp, **b})
    for a in [(z(4, 2, 16, 96),) * 2, (z(4, 2, 24, d),) * 2, (z(4, 2, 8, d),) * 2, (z(4, 2, 2048, d),) * 2]:
        with pytest.raises(E):
            pkg.attn_decode(actx, pkg.KvCache(actx, *a), z(1, 2 * a[0].shape[3]), i(1, 1), i(1))
    for a in [(z(4, 2, 16, d), z(4, 2, 16, d).view(4, 2, 16, d)[:, :1]), (z(4, 2, 16, d), z(4, 2, 16, d, dt=torch.uint8)), (z(4, 2, 16, d, dt=torch.float32),) * 2,
              (z(4, 16, 2, d).transpose(1, 2),) * 2, (z(4, 2, 16, d, dev="cpu"),) * 2, (z(4, 2, 16, d, dt=torch.uint8),) * 2 + (z(3, dt=torch.float32),)]:
        with pytest.raises(E):
            pkg.KvCache(actx, *a)
    # empty batches are no error
    assert pkg.attn_decode(actx, cache, z(0, 4 * d), i(0, 1), i(0)).shape == (0, 4 * d)
    assert pkg.attn_prompt(actx, z(0, 4 * d), z(0, 2 * d), z(0, 2 * d), i(1)).shape == (0, 4 * d)
    assert pkg.kv_append(actx, cache, z(0, 2 * d), z(0, 2 * d), i(0), i(0, 1)) is None
    assert actx.status().code == 0


@gpu
def test_another_current_device_is_refused(pkg, actx):
    """The context says device 0; a copy of it that says 5 stands for a caller that has another device current."""
    import ctypes as C
    other = C.create_string_buffer(64 << 10)
    C.memmove(other, actx.h, 64)
    C.cast(other, C.POINTER(C.c_int32))[0] = 5
    L, cache = pkg.lib(), pkg.KvCache.empty(actx, 2, 16, 1, 64)
    x, i, f = bf16(gen(1), 2, 64), torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(2, 64, device=DEV)
    p, s = x.data_ptr(), actx.stream()
    assert L.dsuf_kv_append(other, s, cache.ref, p, 64, p, 64, 1, i.data_ptr(), 0, i.data_ptr(), 1, 1, None, 0, 0, 0, 0, 0, 0, 0) == -1
    assert L.dsuf_attn_decode(other, s, cache.ref, p, 64, 1, 1, i.data_ptr(), 1, i.data_ptr(), 1.0, 0, p, 64, 0, actx.attn_workspace.data_ptr()) == -1
    assert L.dsuf_attn_prompt(other, s, p, 64, p, 64, p, 64, 2, 1, 1, 64, i.data_ptr(), 1, 1.0, 0, p, 64, 0) == -1
    assert L.dsuf_sample(other, s, f.data_ptr(), 64, 2, 64, 0, 0, 0, 0, f.data_ptr(), i.data_ptr(), 0) == -1
    buf = C.create_string_buffer(512)
    L.dsuf_last_error(other, buf, 512)
    assert b"device 0 is current" in buf.value


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 70, 200])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_hidden_values_that_are_not_finite(pkg, actx, d, window, bad):
    """Values of later tokens of the same sequence, and of tokens that the window has left behind, do not reach a row, whatever they are; those that
    it sees do."""
    g = gen(31)
    lens, hq, hkv = [300, 131], 6, 2
    t = sum(lens)
    q, k, v = bf16(g, t, hq * d), bf16(g, t, hkv * d), bf16(g, t, hkv * d)
    where = [(100, 0, 3), (290, 1, d - 1), (300 + 128, 0, 0), (5, 1, 7)]        # (row, kv head, column)
    for r, h, c in where:
        v[r, h * d + c] = bad
    cu = torch.tensor([0, 300, t], dtype=torch.int32, device=DEV)
    out = pkg.attn_prompt(actx, q, k, v, cu, head_dim=d, window=window)
    clean = v.clone()
    for r, h, c in where:
        clean[r, h * d + c] = 0
    want, _, size = prompt64(q, k, clean, lens, hq, hkv, d, window, d ** -0.5)
    hit = torch.zeros(t, hq * d, dtype=torch.bool, device=DEV)
    for r, h, c in where:
        start, n = (0, 300) if r < 300 else (300, 131)
        last = start + n if window == 0 else min(start + n, r + window)
        for head in range(h * 3, h * 3 + 3):
            hit[r:last, head * d + c] = True
    assert torch.equal(~torch.isfinite(out), hit)
    within(torch.where(hit, torch.zeros_like(out), out), torch.where(hit, 0.0, want), size, terms=2 ** -8 + 2 ** -12)
    # and nothing changes where nothing is hidden: the clean input gives the same bits as before in rows without
    assert actx.status().code == 0


@gpu
def test_a_closed_context_is_refused(pkg, actx):
    c = pkg.Ctx(0)
    cache = pkg.KvCache.empty(c, 2, 16, 1, 64)
    q, i = bf16(gen(1), 1, 64), torch.zeros(1, dtype=torch.int32, device=DEV)
    c.close()
    for call in (lambda: pkg.kv_append(c, cache, q, q, i, i.reshape(1, 1)), lambda: pkg.attn_decode(c, cache, q, i.reshape(1, 1), i),
                 lambda: pkg.attn_prompt(c, q, q, q, torch.zeros(2, dtype=torch.int32, device=DEV), head_dim=64), lambda: pkg.sample(c, q.float(), q[0, :1].float())):
        with pytest.raises(pkg.DsufError):
            call()
