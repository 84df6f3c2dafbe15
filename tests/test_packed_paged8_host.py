"""Packed sequences and 8-bit pages without a GPU: argument checks of the C ABI before any launch, and the Python wrappers' refusals."""
import ctypes as C

import pytest
import torch

import forgetting_transformer as ft
from forgetting_transformer.ops import _lib


def _buffer(n=8192):
    buf = (C.c_char * n)()
    base = C.addressof(buf)
    return buf, base + (-base) % 16


def test_packed_c_abi_checks():
    lib = _lib.load()
    _keep, base = _buffer(1 << 16)
    n = [C.c_int64(-1) for _ in range(3)]
    size = lambda *a: lib.fox_packed_bytes(*a, *(C.byref(x) for x in n))
    assert size(3, 500, 700, 4, 2, 64) == 0 and all(x.value > 0 for x in n)
    room, ws = n[0].value, {"fwd": n[1].value, "bwd": n[2].value}
    assert size(3, 500, 256, 4, 2, 64) == 0 and n[1].value == 0 < n[2].value      # walks of few keys stay whole
    assert size(3, 500, 700, 512, 512, 64) == 0 and n[1].value == n[2].value == 0   # as do those of many heads
    for bad in ((0, 5, 5, 4, 2, 64), (1, 0, 5, 4, 2, 64), (1, 5, 0, 4, 2, 64), (65536, 5, 5, 4, 2, 64), (1, (1 << 30) + 1, 5, 4, 2, 64), (1, 5, 5, 3, 2, 64), (1, 5, 5, 4, 2, 48)):
        assert size(*bad) == -1
    assert lib.fox_packed_bytes(1, 5, 5, 4, 2, 64, None, C.byref(n[0]), C.byref(n[1])) == -1
    big = 1 << 40

    def args(B=3, T=500, N=700, H=4, Hk=2, D=64, dtype=0, q=base, k=base, v=base, o=base, st=256, g=base, cu=base, c=base, lse=base, plan=base, bytes=room, work=base, space=big, d_o=base, dq=base, dk=base,
             dv=base, dg=base, delta=base, dc=base):
        view = lambda p: _lib.View(p, 0, 64, st)
        return _lib.PackedArgs(B, T, N, H, Hk, D, dtype, view(q), view(k), view(v), view(o), g, 4, 1, cu, cu, 1.0, c, lse, plan, bytes, view(d_o), view(dq), view(dk), view(dv), dg, 4, 1,
                               delta, dc, work, space)

    fwd = lambda **k: lib.fox_packed_fwd(C.byref(args(**k)), None)
    bwd = lambda **k: lib.fox_packed_bwd(C.byref(args(**k)), None)
    for call in (fwd, bwd):
        for bad, text in ((dict(B=0), b"positive"), (dict(T=0), b"positive"), (dict(B=70000), b"65535"), (dict(D=48), b"head dim"), (dict(dtype=2), b"dtype"), (dict(H=3), b"multiple"),
                          (dict(Hk=0), b"multiple"), (dict(H=70000, Hk=1), b"65535"), (dict(st=1 << 23), b"2^23"), (dict(st=0), b"2^23"), (dict(c=None), b"c and plan"),
                          (dict(plan=None), b"c and plan"), (dict(bytes=room - 1), b"plan too small"), (dict(space=ws["fwd"] - 1), b"workspace too small"), (dict(work=None), b"workspace too small"), (dict(B=60000, H=100, Hk=100, bytes=1 << 40), b"too many")):
            assert call(**bad) == -1 and text in lib.fox_last_error(), (bad, lib.fox_last_error())
        assert call(q=base + 2) == -2 and call(k=base + 4) == -2 and call(o=base + 8) == -2 and call(plan=base + 4) == -2 and call(work=base + 8) == -2 and call(st=60) == -2 and call(v=None) == -1
    assert bwd(space=ws["bwd"] - 1) == -1
    assert fwd(g=None) == -1 and fwd(cu=None) == -1
    for bad in ("lse", "dg", "delta", "dc", "d_o", "dq", "dk", "dv"):
        assert bwd(**{bad: None}) == -1
    assert lib.fox_packed_fwd(None, None) == -1 and lib.fox_packed_bwd(None, None) == -1


def test_paged8_c_abi_checks():
    lib = _lib.load()
    _keep, base = _buffer()

    def pages(P=8, H=4, Hk=2, S=16, D=64, codes=0, k=base, ks=base + 256, g=base + 512, st=64):
        view = _lib.View(k, 2048, 1024, st)
        return _lib.Pages8(P, H, Hk, S, D, codes, view, view, ks, 2, 1, 1, ks, 2, 1, 1, g, 64, 16, 1)

    def append(T=4, dtype=0, x=base, slots=base + 1024, g=base, **kw):
        v = _lib.View(x, 0, 64, 128)
        return lib.fox_paged8_append(C.byref(_lib.Paged8AppendArgs(pages(**kw), T, dtype, v, v, g, 4, 1, slots)), None)

    def gather(B=2, R=2, W=4, T=8, dtype=0, ends=base, out=base + 2048, table=base, **kw):
        return lib.fox_paged_gather(C.byref(_lib.PagedGatherArgs(pages(**kw), B, R, W, T, dtype, table, W, None, ends, out, out, out)), None)

    def decode(B=2, R=2, W=4, most=0, dtype=0, lengths=base, ws=base + 1024, n=1 << 20, q=base, **kw):
        v = _lib.View(q, 256, 64, 128)
        return lib.fox_paged8_decode(C.byref(_lib.Paged8DecodeArgs(pages(**kw), B, R, W, most, dtype, v, v, base, W, lengths, None, 1.0, ws, n)), None)

    for call in (append, gather, decode):
        for bad, text in ((dict(P=0), b"positive"), (dict(H=3), b"multiple"), (dict(Hk=0), b"multiple"), (dict(S=20), b"page_size"), (dict(D=96), b"head dim"), (dict(codes=3), b"codes"),
                          (dict(dtype=2), b"dtype"), (dict(g=None), b"NULL") if call is not gather else (dict(ks=None), b"scales"), (dict(ks=None), b"scales"), (dict(k=None), b"NULL")):
            assert call(**bad) == -1 and text in lib.fox_last_error(), (bad, lib.fox_last_error())
        assert call(st=72) == -2 and call(k=base + 8) == -2
    assert append(codes=2) == -1 and decode(codes=2) == -1
    assert append(T=0) == -1 and append(T=1 << 28, Hk=4) == -1 and append(slots=None) == -1 and append(x=base + 8) == -2
    assert gather(B=0) == -1 and gather(B=5000) == -1 and gather(R=1) == -1 and gather(W=1 << 27) == -1 and gather(T=0) == -1 and gather(ends=None) == -1 and gather(out=base + 8) == -2
    assert gather(T=(1 << 30) + 1) == -1 and gather(codes=2, st=60) == -2
    assert decode(B=0) == -1 and decode(R=0) == -1 and decode(W=0) == -1 and decode(B=3) == -1 and b"3 rows" in lib.fox_last_error()
    assert decode(W=1 << 27) == -1 and decode(most=-1) == -1 and decode(lengths=None) == -1 and decode(q=base + 4) == -2
    assert decode(W=64, n=16) == -1 and b"workspace" in lib.fox_last_error()
    assert decode(W=64, ws=None) == -1 and decode(W=64, ws=base + 8) == -2
    assert decode(st=1 << 30) == -1 and b"2^32" in lib.fox_last_error()
    n = C.c_int64(-1)
    size = lambda *a: lib.fox_paged8_decode_workspace_bytes(*a, C.byref(n))
    assert size(4, 4, 2, 64, 256) == 0 and n.value == 0
    assert size(4, 4, 2, 64, 4096) == 0 and n.value > 0
    few = n.value
    assert size(4, 40, 2, 64, 4096) == 0 and n.value > few     # a piece has a row of the workspace for every query head
    assert size(4, 4, 3, 64, 4096) == -1 and size(0, 4, 2, 64, 64) == -1 and size(1 << 12, 1 << 12, 1, 64, 64) == -1 and size(4, 4, 2, 48, 64) == -1 and size(4, 4, 2, 64, (1 << 30) + 1) == -1
    assert lib.fox_paged8_decode_workspace_bytes(4, 4, 2, 64, 64, None) == -1
    assert lib.fox_paged8_append(None, None) == -1 and lib.fox_paged_gather(None, None) == -1 and lib.fox_paged8_decode(None, None) == -1


def test_wrapper_refusals():
    x, f, cu = torch.zeros(10, 4, 64).bfloat16(), torch.zeros(10, 4), torch.tensor([0, 10], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.forgetting_attention_packed(x, x, x, f, cu)
    for bad in ((x.float(), x, x, f, cu), (x[0], x, x, f, cu), (x, x[:, :3], x[:, :3], f, cu), (x, x, x[:9], f, cu), (x, x, x, f[:, :3], cu), (x, x, x, f, cu.long()), (x, x[:8], x[:8], f[:8], cu)):
        with pytest.raises(AssertionError):
            ft.forgetting_attention_packed(*bad)
    pages, scales, gates = torch.zeros(4, 2, 16, 64, dtype=torch.int8), torch.ones(4, 2, 1), torch.zeros(4, 4, 16)
    table, n = torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.paged_append_8bit(x[:, :2], x[:, :2], f, pages, pages, scales, scales, gates, torch.arange(10))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.paged_forgetting_attention_8bit(x[:3], pages, pages, scales, scales, gates, table, n)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.paged_gather(pages, pages, gates, table, torch.arange(4, dtype=torch.int32), max_tokens=3, k_scales=scales, v_scales=scales)
    from forgetting_transformer.ops.paged8 import _check_pages
    good = (pages, pages, gates, scales, scales)
    for at, bad in ((0, pages.float()), (1, pages[:3]), (2, gates[:, :3]), (2, gates.double()), (3, scales[:, :1]), (4, None), (0, pages[:, :, :12]), (0, pages[..., :48])):
        with pytest.raises(AssertionError):
            _check_pages(*[bad if i == at or (i == 1 and at == 0 and bad.shape != pages.shape) else t for i, t in enumerate(good)])
    make = dict(num_layers=1, num_heads=4, head_dim=64, num_pages=4, max_requests=2, max_length=32, device="cpu")
    for bad in (dict(cache_dtype=torch.float16), dict(num_kv_heads=2), dict(num_kv_heads=3, cache_dtype=torch.int8), dict(cache_dtype=torch.uint8), dict(num_kv_heads=0, cache_dtype=torch.int8)):
        with pytest.raises(AssertionError):
            ft.PagedFgateCache(**{**make, **bad})
    cache = ft.PagedFgateCache(**make, cache_dtype=torch.float8_e4m3fn, num_kv_heads=2)
    assert cache.key_pages[0].shape == (4, 2, 16, 64) and cache.key_scales[0].shape == (4, 2, 1) and cache.log_fgate_pages[0].shape == (4, 4, 16)
    with pytest.raises(AssertionError, match="prompts"):
        cache.attend_prompts(x, 0)


def test_pages_that_share_elements():
    """What the appends ask of the pages of keys and values: random views of one buffer against the sets of their places, and the layouts that pools have."""
    import random
    from forgetting_transformer.ops import _native
    share = _native.load().share_elements
    rng = random.Random(0)
    base, buf = torch.arange(4000), torch.zeros(4000, dtype=torch.int8)
    seen = [0, 0]
    for _ in range(3000):
        shape = [rng.choice([1, 2, 3, 4]) for _ in range(4)]

        def strides():
            s, at = [0] * 4, 1
            for i in rng.sample(range(4), 4):
                s[i], at = at, at * shape[i] * rng.choice([1, 1, 2, 3]) + rng.choice([0, 0, 1])
            return s
        a = strides()
        b = a if rng.random() < 0.6 else strides()
        if rng.random() < 0.1:
            b[rng.randrange(4)] = rng.randrange(1, 5)        # (rows that may lie on each other)
        first = [rng.randrange(200) for _ in range(2)]
        if any(f + sum((n - 1) * st for n, st in zip(shape, s)) >= 4000 for f, s in zip(first, (a, b))):
            continue
        places = [set(base.as_strided(shape, s, f).flatten().tolist()) for f, s in zip(first, (a, b))]
        want = bool(places[0] & places[1])
        assert share(buf.as_strided(shape, a, first[0]), buf.as_strided(shape, b, first[1])) is want, (shape, a, b, first)
        seen[want] += 1
    assert min(seen) > 200
    P, H, S, D = 64, 4, 16, 64
    for shape, at in (((P, 2, H, S, D), 1), ((P, H, 2, S, D), 2), ((P, H, S, 2, D), 3), ((2, P, H, S, D), 0)):
        kv = torch.zeros(shape, dtype=torch.int8)
        k, v = kv.select(at, 0), kv.select(at, 1)
        assert not share(k, v) and not share(v, k) and share(k, k)
        assert share(k[1:], k[:-1]) and share(k[:, 1:], k[:, :-1]) and share(k[:, :, 1:], k[:, :, :-1])
    kv = torch.zeros(P, 2 * H * S * D, dtype=torch.int8)
    k, v = kv[:, :H * S * D].view(P, H, S, D), kv[:, H * S * D:].view(P, S, H, D).transpose(1, 2)     # of different orders within a page
    assert not share(k, v) and share(k, kv[:, D:D + H * S * D].view(P, S, H, D).transpose(1, 2))
    same = k[:1].expand(P, H, S, D)                                  # (pages that lie on each other)
    assert not share(k, torch.zeros_like(k)) and share(same, same[:, :, :1].expand(P, H, S, D)) and not share(same, v)
    with pytest.raises(RuntimeError, match="one shape"):
        share(k, k[:1])
