"""Argument checks of the cache, attention and sampling entries, without a GPU: the C entries refuse before they touch a device (a zeroed block
stands in for the context, which they only write their message into), the Python mirror before it calls them."""
import ctypes as C
import math
import types

import pytest
import torch

P = 1 << 20          # an aligned address that nothing follows
BAD = -1


@pytest.fixture()
def cctx():
    return C.create_string_buffer(64 << 10)


def cache(pkg, **kw):
    f = dict(k=P, v=P, k_scale=0, v_scale=0, page_stride=2 * 16 * 128, dtype=0, n_pages=4, page_size=16, kv_heads=2, head_dim=128)
    f.update(kw)
    return pkg.KvCacheStruct(*(f[n] for n, _ in pkg.KvCacheStruct._fields_))


def rope(pkg, **kw):
    f = dict(cos=P, sin=P, positions=8, rot=128, off=0, half=0)
    f.update(kw)
    return pkg.RopeStruct(*(f[n] for n, _ in pkg.RopeStruct._fields_))


BAD_CACHES = [dict(dtype=2), dict(head_dim=96), dict(head_dim=256), dict(page_size=8), dict(page_size=24), dict(page_size=2048), dict(page_size=0), dict(kv_heads=0),
              dict(kv_heads=-1), dict(n_pages=0), dict(page_stride=16), dict(page_stride=2 * 16 * 128 + 8), dict(page_stride=-4096), dict(k=0), dict(v=P + 8),
              dict(k_scale=P), dict(dtype=1, k_scale=P + 2)]


def append(pkg, c, ctx, **kw):
    a = dict(k=P, ldk=256, v=P, ldv=256, t=3, pos=P, seq=P, table=P, n_seqs=2, max_pages=4, rope=None, q=P, ldq=512, q_heads=4, q_out=P, ldqo=512, k_out=0, ldko=0)
    a.update(kw)
    r = a["rope"]
    return pkg.lib().dsuf_kv_append(ctx, None, C.byref(c), a["k"], a["ldk"], a["v"], a["ldv"], a["t"], a["pos"], a["seq"], a["table"], a["n_seqs"], a["max_pages"],
                                    C.byref(r) if r is not None else None, a["q"], a["ldq"], a["q_heads"], a["q_out"], a["ldqo"], a["k_out"], a["ldko"])


def test_append_refuses(pkg, cctx):
    for kw in BAD_CACHES:
        assert append(pkg, cache(pkg, **kw), cctx) == BAD, kw
    for kw in [dict(t=-1), dict(n_seqs=-1), dict(max_pages=0), dict(max_pages=1 << 28), dict(seq=0), dict(q_heads=-1), dict(q_heads=5000), dict(ldk=255), dict(ldk=260), dict(ldv=128),
               dict(ldq=511), dict(ldqo=256), dict(ldq=516), dict(k=0), dict(k=P + 8), dict(v=0), dict(pos=0), dict(pos=P + 1), dict(table=0), dict(seq=P + 2), dict(q=0), dict(q_out=0),
               dict(q_out=P + 4), dict(k_out=P, ldko=128), dict(k_out=P + 2, ldko=256)]:
        assert append(pkg, cache(pkg), cctx, **kw) == BAD, kw
    for kw in [dict(rot=0), dict(rot=24), dict(rot=144), dict(off=-8), dict(off=8), dict(rot=64, off=4), dict(cos=0), dict(sin=P + 4), dict(positions=0)]:
        assert append(pkg, cache(pkg), cctx, rope=rope(pkg, **kw)) == BAD, kw
    buf = C.create_string_buffer(512)
    pkg.lib().dsuf_last_error(cctx, buf, 512)
    assert b"rope" in buf.value
    assert append(pkg, cache(pkg), cctx, t=0, k=0, v=0, pos=0, seq=0, table=0, q=0, q_out=0) == 0      # an empty batch
    assert append(pkg, cache(pkg), None) == BAD
    assert pkg.lib().dsuf_kv_append(cctx, None, None, P, 256, P, 256, 1, P, P, P, 1, 1, None, 0, 0, 0, 0, 0, 0, 0) == BAD


def decode(pkg, c, ctx, **kw):
    a = dict(q=P, ldq=512, q_heads=4, b=2, table=P, max_pages=4, lens=P, scale=0.1, window=0, out=P, ldo=512, lse=0, ws=P)
    a.update(kw)
    return pkg.lib().dsuf_attn_decode(ctx, None, C.byref(c), a["q"], a["ldq"], a["q_heads"], a["b"], a["table"], a["max_pages"], a["lens"], a["scale"], a["window"], a["out"],
                                      a["ldo"], a["lse"], a["ws"])


def test_decode_refuses(pkg, cctx):
    for kw in BAD_CACHES:
        assert decode(pkg, cache(pkg, **kw), cctx) == BAD, kw
    for kw in [dict(b=-1), dict(max_pages=0), dict(max_pages=1 << 27), dict(q_heads=3), dict(q_heads=0), dict(q_heads=8192), dict(ldq=256), dict(ldq=514), dict(ldo=511), dict(scale=0.0),
               dict(scale=-0.1), dict(scale=math.nan), dict(scale=math.inf), dict(window=-1), dict(q=0), dict(q=P + 8), dict(out=0), dict(table=0), dict(lens=0), dict(lens=P + 2),
               dict(lse=P + 1), dict(ws=0), dict(ws=P + 8), dict(b=1 << 24, max_pages=1 << 20)]:
        assert decode(pkg, cache(pkg), cctx, **kw) == BAD, kw
    assert decode(pkg, cache(pkg), cctx, b=0, q=0, out=0, table=0, lens=0, ws=0) == 0
    assert decode(pkg, cache(pkg), None) == BAD
    assert pkg.lib().dsuf_attn_workspace_bytes(None) == 0
    assert pkg.lib().dsuf_attn_workspace_init(cctx, None, 0, 1 << 30) == BAD


def prompt(pkg, ctx, **kw):
    a = dict(q=P, ldq=512, k=P, ldk=256, v=P, ldv=256, t=9, hq=4, hkv=2, d=128, cu=P, n=1, scale=0.1, window=0, out=P, ldo=512, lse=0)
    a.update(kw)
    return pkg.lib().dsuf_attn_prompt(ctx, None, a["q"], a["ldq"], a["k"], a["ldk"], a["v"], a["ldv"], a["t"], a["hq"], a["hkv"], a["d"], a["cu"], a["n"], a["scale"], a["window"],
                                      a["out"], a["ldo"], a["lse"])


def test_prompt_refuses(pkg, cctx):
    for kw in [dict(d=96), dict(d=32), dict(hq=3), dict(hkv=0), dict(hq=0), dict(hq=4098, ldq=1 << 20), dict(t=-1), dict(n=-1), dict(ldq=504), dict(ldk=252), dict(ldv=128), dict(ldo=516),
               dict(scale=0.0), dict(scale=math.nan), dict(window=-1), dict(q=0), dict(k=P + 8), dict(v=0), dict(out=P + 2), dict(cu=0), dict(cu=P + 2), dict(lse=P + 3)]:
        assert prompt(pkg, cctx, **kw) == BAD, kw
    assert prompt(pkg, cctx, t=0, q=0, k=0, v=0, out=0, cu=0) == 0 and prompt(pkg, cctx, n=0, cu=0) == 0
    assert prompt(pkg, None) == BAD


def test_prompt_refuses_an_output_in_its_inputs(pkg, cctx):
    row = 512 + 256 + 256 + 512      # q, k, v and the output as columns of one row
    base = dict(ldq=row, ldk=row, ldv=row, ldo=row, q=P, k=P + 1024, v=P + 1536, out=P + 2048)
    text = C.create_string_buffer(512)
    C.c_int.from_buffer(cctx).value = 1 << 20      # (the context's device, never the current one: the good calls go no further than that check)

    def refused(**kw):
        assert prompt(pkg, cctx, **{**base, **kw}) != 0
        pkg.lib().dsuf_last_error(cctx, text, 512)
        return b"share memory" in text.value
    for kw in [dict(out=P), dict(out=P + 1024), dict(out=P + 1536), dict(out=P + 1024 + 496), dict(out=P + 2 * row), dict(out=P, ldo=512), dict(out=P + 16 * row, ldo=520),
               dict(out=P - 16), dict(ldq=512, ldo=512, out=P + 1024 * 8)]:
        assert refused(**kw), kw
    for kw in [{}, dict(out=P + 2048 + 2 * row), dict(out=P + 2 * 9 * row), dict(out=P - 2 * 9 * row), dict(out=P - 1024, ldo=row), dict(ldq=512, out=P + (1 << 16), ldo=512)]:
        assert not refused(**kw), kw


def test_flags_and_offsets_are_refused(pkg, cctx):
    assert append(pkg, cache(pkg), cctx, rope=rope(pkg, rot=16, off=0x7ffffff8)) == BAD      # (their sum passes 32 bits)

    class Neither:
        def __bool__(self):
            raise ValueError("neither")
    ctx = types.SimpleNamespace(torch=torch, device=torch.device("cpu"), index=-1, address=C.addressof(cctx))
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)   # noqa: E731
    with pytest.raises(pkg.DsufError, match="return_lse"):
        pkg.attn_prompt(ctx, z(3, 512), z(3, 256), z(3, 256), z(2, dt=torch.int32), return_lse=Neither())
    with pytest.raises(pkg.DsufError, match="return_logprobs"):
        pkg.sample(ctx, z(3, 9, dt=torch.float32), z(3, dt=torch.float32), return_logprobs=Neither())


def test_sample_refuses(pkg, cctx):
    def call(ctx=cctx, logits=P, ld=100, m=2, n=100, t=0, k=0, p=0, q=0, u=P, ids=P, lp=0):
        return pkg.lib().dsuf_sample(ctx, None, logits, ld, m, n, t, k, p, q, u, ids, lp)
    for kw in [dict(m=-1), dict(n=0), dict(n=(1 << 22) + 1, ld=1 << 23), dict(ld=99), dict(logits=0), dict(u=0), dict(ids=0), dict(ids=P + 1), dict(t=P + 2), dict(lp=P + 3), dict(m=1 << 28),
               dict(ctx=None)]:
        assert call(**kw) == BAD, kw
    assert call(m=0, logits=0, u=0, ids=0) == 0


def test_the_mirror_refuses(pkg, cctx):
    """Shapes, types, devices and strides, on CPU tensors with a stand-in for the context."""
    dev = torch.device("cpu")
    address = C.addressof(cctx)
    space = torch.zeros(16, dtype=torch.uint8)
    ctx = types.SimpleNamespace(torch=torch, device=dev, index=-1, address=address, attn_workspace=space)
    E = pkg.DsufError
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt)   # noqa: E731
    i = lambda *s: z(*s, dt=torch.int32)   # noqa: E731
    for a in [(z(4, 2, 16),) * 2, (z(4, 2, 16, 128, dt=torch.float32),) * 2, (z(4, 2, 16, 128), z(4, 2, 16, 64)), (z(4, 16, 2, 128).transpose(1, 2),) * 2,
              (z(4, 2, 16, 128), z(8, 2, 16, 128)[::2]), (z(4, 2, 16, 128, dt=torch.uint8),) * 2 + (z(2),)]:
        with pytest.raises(E):
            pkg.KvCache(ctx, *a)
    c = pkg.KvCache(ctx, z(8, 2, 16, 128)[::2], z(8, 2, 16, 128)[::2])
    assert c.c.page_stride == 2 * 2 * 16 * 128 and (c.n_pages, c.kv_heads, c.page_size, c.head_dim) == (4, 2, 16, 128)
    good = (z(3, 256), z(3, 256), i(3), i(3, 1))
    for at, bad in [(0, z(3, 256, dt=torch.float16)), (0, z(256, 3).t()), (0, z(3, 128)), (0, z(768)), (0, z(2, 256).as_strided((2, 256), (128, 1))), (0, None), (0, 3), (1, z(2, 256)),
                    (2, i(4)), (2, i(6)[::2]), (2, i(3, 1)), (2, z(3, dt=torch.int64)), (3, i(3)), (3, i(3, 4)[:, :2]), (3, z(3, 1))]:
        with pytest.raises(E, match="kv_append"):
            pkg.kv_append(ctx, c, *(bad if n == at else x for n, x in enumerate(good)))
    for kw in [dict(seq=i(2)), dict(rope=(1, 2)), dict(rope=3), dict(rope=(z(4, 64), z(4, 64), 0)), dict(rope=(z(4, 64, dt=torch.float32), z(4, 32, dt=torch.float32), 0)),
               dict(rope=(z(4, 64, dt=torch.float32),) * 2 + ("x",)), dict(rope=(z(4, 64, dt=torch.float32),) * 2 + (1 << 40,)), dict(q=z(3, 100)), dict(q=z(3, 0)), dict(q=z(3, 256), q_out=z(3, 128)),
               dict(k_out=z(2, 256))]:
        with pytest.raises(E):
            pkg.kv_append(ctx, c, *good, **kw)
    other = types.SimpleNamespace(**vars(ctx))
    with pytest.raises(E, match="another context"):
        pkg.attn_decode(other, c, z(1, 512), i(1, 1), i(1))
    with pytest.raises(E, match="another context"):
        pkg.kv_append(other, c, *good)
    for a, kw in [((z(1, 384), i(1, 1), i(1)), {}), ((z(1, 512), i(2, 1), i(1)), {}), ((z(1, 512), i(1, 1), i(2)), {}), ((z(1, 512), i(1, 1), i(1)), dict(scale="x")),
                  ((z(1, 512), i(1, 1), i(1)), dict(window=1.5)), ((z(1, 512), i(1, 1), i(1)), dict(window=1 << 40)), ((z(1, 512), i(1, 1), i(1)), dict(workspace=z(3)))]:
        with pytest.raises(E, match="attn_decode"):
            pkg.attn_decode(ctx, c, *a, **kw)
    for a, kw in [((z(3, 512), z(3, 256), z(3, 256), i(2)), dict(head_dim=100)), ((z(3, 500), z(3, 256), z(3, 256), i(2)), {}), ((z(3, 512), z(3, 256), z(3, 128), i(2)), {}),
                  ((z(3, 512), z(3, 256), z(3, 256), i(0)), {}), ((z(3, 512), z(3, 256), z(3, 256), i(2)), dict(out=z(3, 256))),
                  ((z(3, 512), z(3, 256), z(3, 256), i(2)), dict(lse=z(3, 4))), ((z(3, 512), z(3, 256), z(3, 256), i(2)), dict(head_dim="a"))]:
        with pytest.raises(E, match="attn_prompt"):
            pkg.attn_prompt(ctx, *a, **kw)
    f = z(3, dt=torch.float32)
    for a, kw in [((z(3, 9), f), {}), ((z(3, 9, dt=torch.float32), f[:2]), {}), ((z(9, 3, dt=torch.float32).t(), f), {}), ((z(3, 9, dt=torch.float32), f), dict(top_k=f)),
                  ((z(3, 9, dt=torch.float32), f), dict(ids=f)), ((z(3, 9, dt=torch.float32), f), dict(logprobs=i(3)))]:
        with pytest.raises(E, match="sample"):
            pkg.sample(ctx, *a, **kw)
    with pytest.raises(TypeError):
        pkg.hostcall().sample(1, 2)
    # a single row's stride says nothing; an empty batch is no error and touches nothing
    assert pkg.kv_append(ctx, c, z(0, 256), z(0, 256), i(0), i(0, 1), q=z(0, 512)).shape == (0, 512)
    out, lse = pkg.attn_prompt(ctx, z(0, 512), z(0, 256), z(0, 256), i(1), return_lse=True)
    assert out.shape == (0, 512) and lse.shape == (0, 4)
    ids, lp = pkg.sample(ctx, z(0, 9, dt=torch.float32), f[:0], return_logprobs=True)
    assert ids.dtype == torch.int32 and lp.shape == (0,)
    mine = z(0, 512)
    assert pkg.attn_prompt(ctx, z(0, 512), z(0, 256), z(0, 256), i(1), out=mine) is mine
