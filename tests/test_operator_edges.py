"""Calls at the edges of what the cache, attention and sampling entries document: what they refuse before anything reaches the GPU (on CPU tensors, with a
zeroed block in the context's place), and rows, values and streams that the larger tests do not meet."""
import ctypes as C
import math
import os
import types

import pytest
import torch

import test_kv_attention as A

gpu = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture()
def hctx():
    """A stand-in for a context, on the CPU: the entries check their arguments against it and get no further."""
    block = C.create_string_buffer(64 << 10)
    return types.SimpleNamespace(torch=torch, device=torch.device("cpu"), index=-1, address=C.addressof(block), block=block,
                                 attn_workspace=torch.zeros(16, dtype=torch.uint8))


@pytest.fixture(scope="module")
def ectx(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = pkg.Ctx(0, pdl=os.environ.get("DSUF_TEST_PDL", "0") == "1")
    yield c
    c.close()


def i32(*v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def z(*shape, dt=torch.bfloat16):
    return torch.zeros(*shape, dtype=dt)


# ------------------------------------------------------------------ the cache's description
def test_pages_that_overlap_are_refused(pkg, hctx):
    """A page stride below a page's size would make the pages' addresses run past the tensor."""
    page = 2 * 16 * 128
    for k in (z(1, 2, 16, 128).expand(1000, 2, 16, 128), z(4 * page).as_strided((4, 2, 16, 128), (page - 16, 2048, 128, 1)),
              z(4 * page).as_strided((4, 2, 16, 128), (2048, 2048, 128, 1))):
        with pytest.raises(pkg.DsufError, match="KvCache"):
            pkg.KvCache(hctx, k, k)
    with pytest.raises(pkg.DsufError, match="KvCache"):
        pkg.KvCache(hctx, z(4, 2, 16, 128), z(1, 2, 16, 128).expand(4, 2, 16, 128))
    # one page has no stride; pages that touch or lie apart are theirs
    one = pkg.KvCache(hctx, z(1, 2, 16, 128).expand(1, 2, 16, 128), z(1, 2, 16, 128))
    assert one.c.page_stride == page and one.c.n_pages == 1
    assert pkg.KvCache(hctx, z(3, 2, 16, 128), z(3, 2, 16, 128)).c.page_stride == page


@pytest.mark.parametrize("shape", [(4, 0, 16, 128), (4, 2, 16, 0), (0, 2, 16, 128), (4, 2, 0, 128)])
def test_empty_caches_are_refused(pkg, shape):
    """In a process of its own: a division by the number of heads or columns would end it."""
    import subprocess
    import sys
    code = f"""
import ctypes as C, types, torch, sys
sys.path.insert(0, {os.path.dirname(os.path.dirname(os.path.abspath(__file__)))!r})
from __graft_entry__ import load_package
pkg = load_package()
block = C.create_string_buffer(64 << 10)
ctx = types.SimpleNamespace(torch=torch, device=torch.device("cpu"), index=-1, address=C.addressof(block), attn_workspace=torch.zeros(16, dtype=torch.uint8))
b, i = torch.bfloat16, torch.int32
n, h, p, d = {shape}
try:
    pkg.KvCache(ctx, torch.zeros(n, h, p, d, dtype=b), torch.zeros(n, h, p, d, dtype=b))
except pkg.DsufError:
    print("cache refused")
# the native entries by themselves, over a description that has not been checked
c = types.SimpleNamespace(ctx=ctx, s=pkg.KvCacheStruct(1 << 20, 1 << 20, 0, 0, n * h * p * d, 0, n, p, h, d))
c.address = C.addressof(c.s)
for call in (lambda: pkg.attn_decode(ctx, c, torch.zeros(1, 512, dtype=b), torch.zeros(1, 1, dtype=i), torch.zeros(1, dtype=i)),
             lambda: pkg.kv_append(ctx, c, torch.zeros(1, h * d, dtype=b), torch.zeros(1, h * d, dtype=b), torch.zeros(1, dtype=i), torch.zeros(1, 1, dtype=i),
                                   q=torch.zeros(1, 512, dtype=b))):
    try:
        call()
    except pkg.DsufError:
        print("call refused")
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])
    assert r.stdout.split("\n")[:3] == ["cache refused", "call refused", "call refused"], r.stdout


# ------------------------------------------------------------------ the sampler's clusters
def test_no_peer_memory_before_the_cluster_has_started(pkg):
    """A CTA may touch another's shared memory only once that one is known to run, and whether it was is no result that a test could see: the kernel's
    text has a completed cluster barrier ahead of the first such access."""
    import re
    with open(os.path.join(os.path.dirname(pkg.__file__), "csrc", "sample.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index("sample_kernel(const SampleArgs"):]
    touches = re.search(r"in_cta\(|ld_cluster_u32\(|share_bins\(|\.list\(|\.limit\(|fetch_list\(", body).start()
    assert re.search(r"cluster_wait\(\)|cluster_barrier\(\)", body).start() < touches
    assert body.index("cluster_arrive()") < touches or body.index("cluster_barrier()") < touches


# ------------------------------------------------------------------ values that are not finite
@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hq,hkv,lens", [(7, 1, [500, 1, 33, 9]), (12, 1, [2600, 70, 17, 5]), (2, 2, [40] * 400)])
def test_decode_over_infinite_values(pkg, ectx, d, hq, hkv, lens):
    """A visible infinity makes its column infinite, infinities of both signs or a NaN make it NaN, and no other column changes."""
    cache, q, table, n = A.decode_inputs(pkg, ectx, 91 + d, lens, hq, hkv, d, 16, False)
    q = (q * 0.25).contiguous()                # (weights between 2^-20 and 1: none is rounded to nothing)
    clean = pkg.attn_decode(ectx, cache, q, table, n)
    place = lambda i, j: (table[i, j // 16].long(), 0, j % 16)   # noqa: E731
    want = clean.clone().reshape(len(lens), hq, d)
    heads = hq // hkv
    for i, j, c, x in ((0, 3, 5, math.inf), (0, 8, 6, -math.inf), (2, 3, 0, -math.inf), (2, 16, 0, -math.inf), (2, 4, d - 1, math.inf), (2, 5, d - 1, -math.inf), (3, 2, 9, math.nan)):
        cache.v[(*place(i, j), c)] = x
        want[i, :heads, c] = x if x != -math.inf or c != d - 1 else math.nan
    out = pkg.attn_decode(ectx, cache, q, table, n).reshape(want.shape)
    torch.cuda.synchronize()
    assert ectx.status().code == 0
    assert torch.equal(torch.isnan(out), torch.isnan(want)) and torch.equal(out.nan_to_num(0, 1e38, -1e38), want.nan_to_num(0, 1e38, -1e38))


@gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_scores_below_all_others(pkg, ectx, fp8):
    """Scores that, times log2(e), lie between -3.4e38 and -3e38: equal ones give the plain mean of the visible values, and their own lse."""
    g = A.gen(62)
    d, n = 64, 300
    c = -3.46e36                               # (times 64 columns: -2.21e38, times log2(e): -3.19e38)
    q = torch.ones(n, 2 * d, dtype=torch.bfloat16, device=DEV)
    k, v = torch.full((n, d), c, dtype=torch.float32, device=DEV).bfloat16(), A.bf16(g, n, d)
    score = 64 * float(k[0, 0])
    assert -3.4e38 < score * math.log2(math.e) < -3e38
    mean = lambda rows: (rows.mean(0).expand(2, d), rows.abs().mean(0).expand(2, d))   # noqa: E731
    if not fp8:
        for window in (0, 50):
            out, lse = pkg.attn_prompt(ectx, q, k, v, i32(0, n), head_dim=d, scale=1.0, window=window, return_lse=True)
            for r in (0, 1, 49, 128, 299):
                want, size = mean(v.double()[max(0, r + 1 - window) if window else 0: r + 1])
                A.within(out[r].reshape(2, d), want, size, terms=2 ** -8 + 2 ** -12)
            # three fp32 roundings: of the sum of 64 equal terms, none; of its product with log2(e) and of that with ln(2), and of both constants
            assert ((lse.double() - score).abs() <= 2 ** -21 * abs(score)).all()
    scale = torch.tensor([float(k[0, 0]) / -448], device=DEV)
    cache = pkg.KvCache.empty(ectx, 20, 16, 1, d, fp8, *((scale, scale * 0 + 0.05) if fp8 else ()))
    pos = torch.arange(n, dtype=torch.int32, device=DEV)
    table = torch.arange(19, dtype=torch.int32, device=DEV)[None]
    pkg.kv_append(ectx, cache, k, v, pos, table, seq=torch.zeros_like(pos))
    seen = A.cache64(cache)[1][:19].transpose(1, 2).reshape(-1, d)[:n]
    for window in (0, 50):
        want, size = mean(seen[n - window if window else 0:])
        out, lse = pkg.attn_decode(ectx, cache, q[:1], table, pos[-1:] + 1, scale=1.0, window=window, return_lse=True)
        A.within(out.reshape(2, d), want, size, terms=2 ** -8 + 2 ** -12)
        assert ((lse.double() - score).abs() <= 2 ** -20 * abs(score)).all()
    assert ectx.status().code == 0


@gpu
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [0, 3000])
def test_hidden_values_in_a_long_prompt(pkg, ectx, d, window):
    """Values that are not finite near a long prompt's end: the rows of their tile that do not see them are computed from what they see, every other output keeps
    its bits."""
    n, hq, hkv = 20000, 4, 2
    g = A.gen(131)
    q, k, v = A.bf16(g, n, hq * d), A.bf16(g, n, hkv * d), A.bf16(g, n, hkv * d)
    cu = i32(0, n)
    clean = pkg.attn_prompt(ectx, q, k, v, cu, head_dim=d, window=window).reshape(n, hq, d)
    bad = v.clone()
    where = [(19990, 0, 3, math.nan), (19990, 1, d - 1, math.inf), (19969, 1, 0, -math.inf), (10000, 1, 40, math.nan)]         # the last tile begins at 19968
    want = clean.clone()
    by_other_means = torch.zeros(n, hq, d, dtype=torch.bool, device=DEV)
    for r, h, c, x in where:
        bad[r, h * d + c] = x
        last = min(n, r + window) if window else n
        heads = slice(2 * h, 2 * h + 2)
        want[r:last, heads, c] = x
        by_other_means[r // 128 * 128: r, heads, c] = True
        if window and last < n:      # (up to the last tile of rows whose first row still sees a key of this key's tile, and so meets the whole tile)
            by_other_means[last: ((r // 128 * 128 + 127 + window - 1) // 128 + 1) * 128, heads, c] = True
    out = pkg.attn_prompt(ectx, q, k, bad, cu, head_dim=d, window=window).reshape(n, hq, d)
    torch.cuda.synchronize()
    assert ectx.status().code == 0
    same = lambda x: torch.where(by_other_means, torch.zeros_like(x), x).nan_to_num(7e30, 8e30, 9e30)   # noqa: E731
    assert torch.equal(same(out), same(want))
    for r in sorted(set(by_other_means.any(2).any(1).nonzero().flatten().tolist())):
        lo = max(0, r + 1 - window) if window else 0
        for h in range(hq):
            cols = by_other_means[r, h].nonzero().flatten()
            if len(cols) == 0:
                continue
            kk, vv = (x[lo: r + 1].double().reshape(-1, hkv, d)[:, h // 2] for x in (k, v))
            p = torch.softmax(kk @ q[r].double().reshape(hq, d)[h] * d ** -0.5, 0)
            A.within(out[r, h, cols], (p @ vv)[cols], (p @ vv.abs())[cols], terms=2 ** -8 + 2 ** -12)


@gpu
@pytest.mark.parametrize("window", [0, 70])
def test_hidden_nan_beside_a_visible_infinity(pkg, ectx, window):
    """The rows that see the infinity and not the NaN in the same column have an infinity there."""
    d, n = 64, 300
    g = A.gen(132)
    q, k, v = A.bf16(g, n, 2 * d), A.bf16(g, n, d), A.bf16(g, n, d)
    for r, c, x in ((130, 5, math.inf), (200, 5, math.nan), (129, 6, -math.inf), (250, 6, math.inf), (10, 7, math.inf), (40, 7, math.nan)):
        v[r, c] = x
    out = pkg.attn_prompt(ectx, q, k, v, i32(0, n), head_dim=d, window=window).reshape(n, 2, d)
    for c in (5, 6, 7):
        for r in range(n):
            seen = v[max(0, r + 1 - window) if window else 0: r + 1, c].float()
            odd = seen[~torch.isfinite(seen)].tolist()
            for x in out[r, :, c].tolist():
                if not odd:
                    assert math.isfinite(x), (r, c, x)
                elif len(set(odd)) > 1 or math.isnan(odd[0]):
                    assert math.isnan(x), (r, c, x)
                else:
                    assert x == odd[0], (r, c, x)
    assert ectx.status().code == 0


# ------------------------------------------------------------------ outputs that lie in inputs
P = 1 << 24          # an aligned address that nothing follows


def shares(pkg, block, rc):
    text = C.create_string_buffer(512)
    pkg.lib().dsuf_last_error(block, text, 512)
    assert rc != 0           # (the calls that pass the check end at the next one: the stand-in's device is never the current one)
    return b"share no memory" in text.value


@pytest.fixture()
def cblock():
    block = C.create_string_buffer(64 << 10)
    C.c_int.from_buffer(block).value = 1 << 20
    return block


ROW = 4 * 128 + 2 * 128 + 2 * 128        # q, k and v of a token beside each other


def test_append_refuses_outputs_in_its_inputs(pkg, cblock):
    cache = pkg.KvCacheStruct(P >> 4, P >> 4, 0, 0, 2 * 16 * 128, 0, 4, 16, 2, 128)

    def refused(t=9, q=P, k=P + 1024, v=P + 1536, ld=ROW, q_out=P + (1 << 20), ldqo=512, k_out=0, ldko=0):
        return shares(pkg, cblock, pkg.lib().dsuf_kv_append(cblock, None, C.byref(cache), k, ld, v, ld, t, P - 4096, P - 4096, P - 4096, 2, 4, None, q, ld, 4, q_out, ldqo,
                                                           k_out, ldko))
    for kw in [dict(q_out=P + 16, ldqo=ROW), dict(q_out=P, ldqo=512), dict(q_out=P + 2 * ROW, ldqo=ROW), dict(q_out=P + 1024, ldqo=ROW), dict(q_out=P + 1536, ldqo=ROW),
               dict(q_out=P - 1008, ldqo=512, t=1), dict(q_out=P + 1024 * 4, ldqo=520),
               dict(k_out=P + 1024 + 16, ldko=ROW), dict(k_out=P + 1024, ldko=256), dict(k_out=P + 1536, ldko=ROW), dict(k_out=P, ldko=ROW), dict(k_out=P + 1024 + 2 * ROW, ldko=ROW),
               dict(k_out=P + (1 << 20), ldko=256), dict(k_out=P + (1 << 20) + 512, ldko=512)]:
        assert refused(**kw), kw
    for kw in [{}, dict(q_out=P, ldqo=ROW), dict(q_out=P, ldqo=512, t=1), dict(k_out=P + 1024, ldko=ROW), dict(k_out=P + 1024, ldko=256, t=1), dict(q_out=P, ldqo=ROW, k_out=P + 1024, ldko=ROW),
               dict(k_out=P + (2 << 20), ldko=256), dict(q_out=P + 2 * 9 * ROW, ldqo=512), dict(q_out=P - 2 * 9 * 512, ldqo=512),
               dict(q=P, k=P + 1024, v=P + 1536, ld=2 * ROW, q_out=P + 2 * ROW, ldqo=2 * ROW)]:
        assert not refused(**kw), kw


def test_decode_refuses_outputs_in_its_inputs(pkg, cblock):
    cache = pkg.KvCacheStruct(P >> 4, P >> 4, 0, 0, 2 * 16 * 128, 0, 4, 16, 2, 128)

    def refused(b=9, q=P, ldq=512, out=P + (1 << 20), ldo=512, lse=0):
        return shares(pkg, cblock, pkg.lib().dsuf_attn_decode(cblock, None, C.byref(cache), q, ldq, 4, b, P - 4096, 4, P - 4096, 0.1, 0, out, ldo, lse, P + (1 << 22)))
    for kw in [dict(out=P + 16), dict(out=P + 1024), dict(out=P, ldo=520), dict(out=P - 1008), dict(out=P + 1008, b=1), dict(out=P, ldq=1024), dict(ldq=1024, ldo=1024, out=P + 1008),
               dict(lse=P), dict(lse=P + 9 * 1024 - 4), dict(lse=P - 9 * 16 + 4), dict(lse=P + (1 << 20) + 1024), dict(lse=P + 1040, ldq=1024, ldo=1024, out=P + 1024)]:
        assert refused(**kw), kw
    for kw in [{}, dict(out=P), dict(out=P, b=1, ldo=520), dict(out=P + 9 * 1024), dict(out=P - 9 * 1024), dict(ldq=1024, ldo=1024, out=P + 1024), dict(lse=P + 9 * 1024),
               dict(lse=P - 9 * 16), dict(lse=P + 1024, ldq=1024, b=1), dict(lse=P + 1024, ldq=1024)]:
        assert not refused(**kw), kw


def test_prompt_refuses_an_lse_in_its_inputs(pkg, cblock):
    def refused(t=9, ld=ROW, out=P + (1 << 20), ldo=512, lse=0):
        return shares(pkg, cblock, pkg.lib().dsuf_attn_prompt(cblock, None, P, ld, P + 1024, ld, P + 1536, ld, t, 4, 2, 128, P - 4096, 1, 0.1, 0, out, ldo, lse))
    for kw in [dict(lse=P), dict(lse=P + 1024), dict(lse=P + 1536 + 4), dict(lse=P + 9 * 2 * ROW - 4), dict(lse=P - 9 * 16 + 4), dict(lse=P + (1 << 20)), dict(lse=P + (1 << 20) + 9 * 1024 - 4)]:
        assert refused(**kw), kw
    for kw in [{}, dict(lse=P + 9 * 2 * ROW), dict(lse=P - 9 * 16), dict(lse=P + (1 << 20) + 9 * 1024), dict(ld=2 * ROW, lse=P + 2 * ROW)]:
        assert not refused(**kw), kw


# ------------------------------------------------------------------ the workspace
def test_workspace_init_refuses_another_current_device(pkg, cblock):
    """The stand-in's device is never the current one.  (Its zeroed number of SMs asks for no bytes, so a memset that is let through does nothing.)"""
    assert pkg.lib().dsuf_attn_workspace_bytes(cblock) == 0
    assert pkg.lib().dsuf_attn_workspace_init(cblock, None, P, 0) != 0
    text = C.create_string_buffer(512)
    pkg.lib().dsuf_last_error(cblock, text, 512)
    assert text.value.startswith(b"attn_workspace_init"), text.value


def test_no_new_workspace_under_capture(pkg):
    """Its zeroing would only be recorded, and a call before the graph's first replay would find arbitrary counters."""
    done = []
    t = types.SimpleNamespace(uint8=torch.uint8, empty=lambda *a, **k: done.append("empty") or torch.zeros(8, dtype=torch.uint8),
                              cuda=types.SimpleNamespace(is_current_stream_capturing=lambda: True, current_stream=lambda d: None))
    ctx = types.SimpleNamespace(torch=t, h=None, device=torch.device("cpu"), index=0, check=lambda rc: None, stream=lambda: None)
    with pytest.raises(pkg.DsufError, match="captur"):
        pkg.Ctx.new_attn_workspace(ctx)
    assert not done


# ------------------------------------------------------------------ scores of very different sizes
@gpu
@pytest.mark.parametrize("d,hq,hkv,lens", [(128, 7, 1, [300, 40]), (64, 24, 2, [77, 900]), (128, 3, 1, [50] * 400)])
def test_a_head_is_alone_with_its_scale(pkg, ectx, d, hq, hkv, lens):
    """Over an e4m3 cache queries are brought into fp16's range: one head's size does not touch another's result."""
    cache, q, table, n = A.decode_inputs(pkg, ectx, 41, lens, hq, hkv, d, 16, True)
    q = q.reshape(len(lens), hq, d).clone()
    q[:, 1] *= 2.0 ** 60
    q[:, 2] *= 2.0 ** -60
    out, lse = pkg.attn_decode(ectx, cache, q.reshape(len(lens), -1), table, n, return_lse=True)
    torch.cuda.synchronize()
    assert ectx.status().code == 0
    want, wl, size = A.decode64(cache, q.reshape(len(lens), -1), table, lens, 0, d ** -0.5)
    keep = [h for h in range(hq) if h != 1]         # (head 1: all weight on one key, but for ties within its scores' rounding)
    pick = lambda x: x.reshape(len(lens), hq, d)[:, keep]   # noqa: E731
    A.within(pick(out), pick(want), pick(size), terms=2 ** -8 + 2 ** -12)
    assert ((lse.double() - wl)[:, keep].abs() <= 2 ** -12 + 2 ** -22 * wl[:, keep].abs()).all()


# ------------------------------------------------------------------ sizes that the waits' limit would not cover
def test_prompt_refuses_more_sequences_than_its_walk_is_made_for(pkg, cblock):
    """A CTA looks for its next tiles in steps of 32 sequences and one level of lengths; at least every other level has a pair, and a CTA gets one of 148, so
    it takes at most 296 n / 32 steps of about 1000 cycles, which other warps' waits of 4e9 cycles have to cover."""
    limit = 1 << 18
    assert 296 * limit / 32 * 1000 < 4e9

    def call(n):
        rc = pkg.lib().dsuf_attn_prompt(cblock, None, P, ROW, P + 1024, ROW, P + 1536, ROW, 9, 4, 2, 128, P - 4096, n, 0.1, 0, P + (1 << 20), 512, 0)
        text = C.create_string_buffer(512)
        pkg.lib().dsuf_last_error(cblock, text, 512)
        assert rc != 0
        return b"n_seqs" in text.value
    assert call(limit + 1) and call(0x7fffffff) and not call(limit)


def test_sample_refuses_outputs_in_its_inputs(pkg, cblock):
    """A setting's own column may receive the result (each row reads its settings first); nothing else may be shared."""
    far = P + (1 << 22)

    def refused(logits=P, ld=100, m=5, n=100, t=far, k=far + 64, p=far + 128, q=far + 192, u=far + 256, ids=far + 320, lp=far + 384):
        return shares(pkg, cblock, pkg.lib().dsuf_sample(cblock, None, logits, ld, m, n, t, k, p, q, u, ids, lp))
    for kw in [dict(ids=P), dict(lp=P + 4 * 499), dict(ids=P - 4), dict(ids=far + 68), dict(lp=far + 252), dict(lp=far + 320), dict(lp=far + 324), dict(lp=far + 4), dict(ids=far - 16),
               dict(ids=P + 400, ld=101)]:
        assert refused(**kw), kw
    for kw in [{}, dict(ids=far + 64), dict(lp=far + 256), dict(lp=far), dict(lp=0), dict(t=0, k=0, p=0, q=0), dict(ids=P + 2000), dict(ids=P - 20), dict(ids=P + 400, ld=200), dict(ids=far + 44)]:
        assert not refused(**kw), kw


def test_append_refuses_a_place_for_queries_it_was_not_given(pkg, hctx):
    cache = pkg.KvCache(hctx, z(4, 2, 16, 128), z(4, 2, 16, 128))
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(pkg.DsufError, match="q_out"):
        pkg.kv_append(hctx, cache, z(3, 256), z(3, 256), i, i.reshape(3, 1), q_out=z(3, 512))


@gpu
@pytest.mark.parametrize("scale", [1.0, 20.0])
def test_large_scores_within_their_own_rounding(pkg, ectx, scale):
    """Scores of thousands and tens of thousands that grow along the context.  A score is a sum of d products in fp32, in the tensor core at worst cut and not rounded
    (2^-23 each time), times the scale and log2(e) (2^-22): it is off by at most E = (d + 2) 2^-23 scale sum |q k|.  So lse is off by E and its own rounding, a row's
    weights by factors between exp(-2 E) and exp(2 E), and where all weights but the largest add up to r, the output by no more than 2 r exp(2 E)
    of the largest value."""
    g = A.gen(21)
    d, n, hq = 128, 700, 2
    q, k, v = A.bf16(g, n, hq * d), A.bf16(g, n, d), A.bf16(g, n, d)
    k *= (1.0 + torch.arange(n, device=DEV)[:, None] * 0.2).to(torch.bfloat16)
    cu = i32(0, n)
    out, lse = pkg.attn_prompt(ectx, q, k, v, cu, scale=scale, return_lse=True)
    cache = pkg.KvCache.empty(ectx, 44, 16, 1, d)
    table = torch.arange(44, dtype=torch.int32, device=DEV).reshape(1, 44)
    pkg.kv_append(ectx, cache, k, v, torch.arange(n, dtype=torch.int32, device=DEV), table, seq=torch.zeros(n, dtype=torch.int32, device=DEV))
    lens = torch.arange(1, n + 1, dtype=torch.int32, device=DEV)
    out1, lse1 = pkg.attn_decode(ectx, cache, q, table.repeat(n, 1), lens, scale=scale, return_lse=True)
    torch.cuda.synchronize()
    assert ectx.status().code == 0
    want, wl, size = A.prompt64(q, k, v, [n], hq, 1, d, 0, scale)
    q64, k64 = q.double().reshape(n, hq, d), k.double()
    hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
    sharp = 0
    for h in range(hq):
        s = (q64[:, h] @ k64.T * scale).masked_fill(hidden, -math.inf)
        e = ((q64[:, h].abs() @ k64.abs().T) * scale).masked_fill(hidden, 0).amax(1) * (d + 2) * 2 ** -23
        top = s.amax(1, keepdim=True)
        r = torch.exp(s - top).sum(1) - 1
        off = torch.minimum(2 * r * torch.exp(2 * e), torch.full_like(r, 4.0)) * v.double().abs().amax()
        sharp += (off < 2 ** -6).sum().item()
        for o, l in ((out, lse), (out1, lse1)):
            assert ((l[:, h].double() - wl[:, h]).abs() <= e + 2 ** -12 + 2 ** -22 * wl[:, h].abs()).all()
            got, w, z = (x.reshape(n, hq, d)[:, h] for x in (o.double(), want, size))
            assert ((got - w).abs() <= 2 ** -8 * w.abs() + (2 ** -8 + 2 ** -12) * z + off[:, None]).all()
    assert sharp > n * hq / 2             # (most rows are compared closely)


# ------------------------------------------------------------------ the prompt kernel's end
def test_no_copies_or_products_outlive_the_prompt_kernel(pkg):
    """After a wait that has run out a CTA still frees its memory: its text has waits for the copies and the products that it has issued on every way to the
    end, and copies stop at the first such wait.  (The waits cannot run out in a test: nothing that could make them is reachable from outside.)"""
    import re
    with open(os.path.join(os.path.dirname(pkg.__file__), "csrc", "attn_prompt.cu")) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    body = text[text.index("attn_prompt_kernel(const"):]
    body = body[:body.index("tmem_dealloc")]
    producer = body[body.index("if (warp == 8) {", body.index("PromptWalk walk(a)")):body.index("else if (warp >= 9)")]
    issuer = body[body.index("else if (warp >= 9)"):body.index("const uint32_t lanes")]
    for part, issued, waits in ((producer, "tma_2d_nh", ("mbar_wait(&kv_full", "mbar_wait(&q_full")), (issuer, "pa_mma_ts", ("tc_commit(&drained", "mbar_wait(&drained"))):
        for w in waits:
            assert part.rindex(w) > part.rindex(issued), w
    for m in re.finditer("tma_2d_nh", producer):
        assert "warp_elect() && !dead" in producer[max(0, m.start() - 600):m.start()]
    # the phase that the last of n copies into ring slot s completes, counted copy by copy
    for stages in (4, 8):
        for n in range(1, 40):
            fills = [0] * stages
            for i in range(n):
                fills[i % stages] += 1
            for s in range(min(n, stages)):
                assert (n - 1 - s) // stages % 2 == (fills[s] - 1) % 2


@gpu
def test_prompts_of_nothing(pkg, ectx):
    """Sequences without rows: nothing is written, and the next call finds everything in order."""
    q = A.bf16(A.gen(5), 300, 128)
    out, lse = torch.full_like(q, 3.0), torch.full((300, 1), 3.0, device=DEV)
    for cu in (i32(0, 0), i32(0, 0, 0, 0), i32(300, 300), i32(7, 7, 7)):
        pkg.attn_prompt(ectx, q, q, q, cu, out=out, lse=lse)
        torch.cuda.synchronize()
        assert (out == 3.0).all() and (lse == 3.0).all() and ectx.status().code == 0
    pkg.attn_prompt(ectx, q, q, q, i32(0, 0, 300, 300), out=out, lse=lse)
    want, wl, size = A.prompt64(q, q, q, [0, 300, 0], 1, 1, 128, 0, 128 ** -0.5)
    A.within(out, want, size, terms=2 ** -8 + 2 ** -12)
    assert ectx.status().code == 0


@gpu
@pytest.mark.parametrize("m,n", [(1, 129280), (64, 5000), (300, 70)])
@pytest.mark.parametrize("settings", [dict(), dict(top_k=20, top_p=0.9), dict(top_p=0.7), dict(temperature=0.0), dict(min_p=0.05)])
def test_results_in_the_columns_of_settings(pkg, ectx, m, n, settings):
    """Tokens may replace top_k, and log-probabilities the uniform numbers, row for row."""
    g = A.gen(m + n)
    x, u = torch.empty(m, n, device=DEV).normal_(0, 2, generator=g), torch.rand(m, generator=g, device=DEV)
    x[m // 2] = -math.inf
    kw = {k: torch.full((m,), v, dtype=torch.int32 if k == "top_k" else torch.float32, device=DEV) for k, v in settings.items()}
    kw.setdefault("top_k", torch.zeros(m, dtype=torch.int32, device=DEV))
    ids, lp = pkg.sample(ectx, x, u, return_logprobs=True, **kw)
    got, got_lp = pkg.sample(ectx, x, u, ids=kw["top_k"], logprobs=u, return_logprobs=True, **kw)
    assert got is kw["top_k"] and got_lp is u
    assert torch.equal(got, ids) and torch.equal(got_lp, lp)
