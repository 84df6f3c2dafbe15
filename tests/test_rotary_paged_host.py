"""The position rotation and the pages without a GPU: frequencies, argument checks of the C ABI before any launch, and the Python wrappers' refusals."""
import ctypes as C
import math

import pytest
import torch

import forgetting_transformer as ft
from forgetting_transformer.ops import _lib


def _buffer(n=8192):
    buf = (C.c_char * n)()
    base = C.addressof(buf)
    return buf, base + (-base) % 16


def test_frequencies():
    f = ft.rotary_frequencies(64)
    assert f.dtype == torch.float64 and f.shape == (32,)
    assert f[0] == 1.0 and math.isclose(f[-1].item(), 10000.0 ** (-62 / 64), rel_tol=1e-14)
    assert torch.allclose(ft.rotary_frequencies(64, scaling="linear", factor=4.0), f / 4, rtol=1e-14, atol=0)
    b = ft.rotary_frequencies(64, scaling="base", factor=8.0)
    assert b[0] == 1.0 and math.isclose(b[-1].item(), f[-1].item() / 8.0, rel_tol=1e-12) and (b <= f).all()
    p = ft.rotary_frequencies(64, scaling="parts", factor=4.0, original_length=2048)
    turns = 2048 * f / (2 * math.pi)
    assert torch.equal(p[turns >= 32], f[turns >= 32]) and torch.allclose(p[turns <= 1], f[turns <= 1] / 4, rtol=1e-14, atol=0)
    between = (turns > 1) & (turns < 32)
    assert between.any() and (p[between] < f[between]).all() and (p[between] > f[between] / 4).all() and (p[1:] < p[:-1]).all()
    assert ft.rotary_frequencies(2, scaling="base", factor=3.0).tolist() == [1.0]
    for bad in (dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=16, base=0.0), dict(rotary_dim=16, factor=-1.0), dict(rotary_dim=16, scaling="cubic"),
                dict(rotary_dim=16, scaling="parts", factor=2.0), dict(rotary_dim=16, scaling="parts", original_length=64, slow=4.0, fast=4.0)):
        with pytest.raises(ValueError):
            ft.rotary_frequencies(**bad)


def test_rotary_c_abi_checks():
    lib = _lib.load()
    _keep, base = _buffer()

    def args(D=64, R=64, inter=0, sides=1, dtype=0, B=1, T=2, H=1, x=base, y=base + 1024, st=64, w=None, w_sh=0, freq=base + 2048, dx=None, dw=None,
             ws=None, w1=None):
        view = lambda p: _lib.View(p, 128, 64, st)
        side = lambda weight: _lib.RotarySide(H, view(x), view(y), view(dx), weight)
        return _lib.RotaryArgs(sides, B, T, D, dtype, R, inter, (_lib.RotarySide * 2)(side(w), side(w1)), w_sh, 1e-5, freq, None, 0, 0, 0, dw, ws)

    fwd = lambda **k: lib.fox_rotary_fwd(C.byref(args(**k)), None)
    bwd = lambda **k: lib.fox_rotary_bwd(C.byref(args(**k)), None)
    for bad, text in ((dict(D=48), b"head dim"), (dict(R=24), b"rotary_dim"), (dict(R=0), b"rotary_dim"), (dict(R=80), b"rotary_dim"),
                      (dict(R=7, inter=1), b"rotary_dim"), (dict(sides=3), b"sides"), (dict(dtype=2), b"dtype"), (dict(B=0), b"B and T"), (dict(T=-1), b"B and T"),
                      (dict(B=1 << 20, T=1 << 20), b"2^30"), (dict(B=1 << 9, T=1 << 20, H=1), b"2^34"),
                      (dict(B=1 << 9, T=1 << 20, D=16, R=16, st=16, H=3, sides=2), b"2^34"), (dict(H=0), b"heads"), (dict(x=None), b"x is NULL"), (dict(y=None), b"y is NULL"),
                      (dict(freq=None), b"inv_freq"), (dict(w=base, w_sh=5), b"weight_stride_h"), (dict(sides=2, w=base), b"both sides"),
                      (dict(sides=2, w1=base), b"both sides")):
        assert fwd(**bad) == -1 and text in lib.fox_last_error(), (bad, lib.fox_last_error())
    assert fwd(x=base + 2) == -2 and fwd(y=base + 1026) == -2 and fwd(st=60) == -2 and fwd(w=base + 4) == -2
    assert bwd() == -1 and b"dx is NULL" in lib.fox_last_error()
    assert bwd(dx=base, w=base) == -1 and b"dweight" in lib.fox_last_error()
    assert bwd(dx=base, w=base, dw=base, ws=base + 4) == -2
    assert lib.fox_rotary_fwd(None, None) == -1 and lib.fox_rotary_bwd(None, None) == -1
    n = C.c_int64(0)
    assert lib.fox_rotary_workspace_bytes(4096, 24, 64, 0, C.byref(n)) == 0 and n.value >= 24 * 64 * 4
    assert lib.fox_rotary_workspace_bytes(0, 24, 64, 0, C.byref(n)) == -1 and lib.fox_rotary_workspace_bytes(1, 1, 48, 0, C.byref(n)) == -1
    assert lib.fox_rotary_workspace_bytes(1, 0, 64, 0, C.byref(n)) == -1 and lib.fox_rotary_workspace_bytes(1, 1, 64, 0, None) == -1


def test_page_c_abi_checks():
    lib = _lib.load()
    _keep, base = _buffer()

    def slots(B=2, W=4, P=8, S=16, T=4, lengths=base, out=base + 512, count=base + 256, count_out=base + 768, slots=base + 1024, table=base + 64):
        return lib.fox_page_slots(C.byref(_lib.PageSlotsArgs(B, W, P, S, T, lengths, base + 32, table, W, base + 128, count, slots, base + 1536, base + 2048, base + 2304,
                                                             out, count_out, base + 2560)), None)

    for bad, text in ((dict(B=0), b"positive"), (dict(W=0), b"positive"), (dict(P=0), b"positive"), (dict(B=4097), b"4096"), (dict(S=4), b"page_size"), (dict(S=24), b"page_size"),
                      (dict(S=8192), b"page_size"), (dict(W=1 << 28, S=4096), b"2^30"), (dict(T=-1), b"max_tokens"), (dict(lengths=None), b"NULL"),
                      (dict(slots=None), b"NULL"), (dict(table=None), b"NULL"), (dict(out=base), b"in place"), (dict(count_out=base + 256), b"in place")):
        assert slots(**bad) == -1 and text in lib.fox_last_error(), (bad, lib.fox_last_error())

    def release(B=2, W=4, P=8, S=16, done=base + 32):
        return lib.fox_page_release(C.byref(_lib.PageReleaseArgs(B, W, P, S, base, done, base + 64, W, base + 128, base + 256, base + 512, base + 768)), None)

    for bad, text in ((dict(B=0), b"positive"), (dict(B=5000), b"4096"), (dict(S=12), b"page_size"), (dict(done=None), b"NULL")):
        assert release(**bad) == -1 and text in lib.fox_last_error()

    def pages(P=8, H=2, S=16, D=64, dtype=0, k=base, g=base + 512, st=64):
        view = _lib.View(k, 2048, 1024, st)
        return _lib.Pages(P, H, S, D, dtype, view, view, g, 32, 16, 1)

    def append(T=4, k=base, slots=base + 1024, **kw):
        v = _lib.View(k, 0, 64, 128)
        return lib.fox_paged_append(C.byref(_lib.PagedAppendArgs(pages(**kw), T, v, v, base, 2, 1, slots)), None)

    def decode(B=2, R=2, W=4, most=0, lengths=base, ws=base + 1024, n=1 << 20, q=base, **kw):
        v = _lib.View(q, 128, 64, 128)
        return lib.fox_paged_decode(C.byref(_lib.PagedDecodeArgs(pages(**kw), B, R, W, most, v, v, base, W, lengths, None, 1.0, ws, n)), None)

    for call in (append, decode):
        for bad, text in ((dict(P=0), b"positive"), (dict(H=0), b"positive"), (dict(S=20), b"page_size"), (dict(D=96), b"head dim"), (dict(dtype=2), b"dtype"),
                          (dict(g=None), b"log gates")):
            assert call(**bad) == -1 and text in lib.fox_last_error(), (bad, lib.fox_last_error())
        assert call(k=None) == -1 if call is append else call(q=None) == -1
        assert call(st=60) == -2
    assert append(T=0) == -1 and append(T=1 << 30, H=4) == -1 and append(slots=None) == -1 and append(k=base + 8) == -2
    assert decode(B=0) == -1 and decode(R=0) == -1 and decode(W=0) == -1 and decode(B=3) == -1 and b"3 rows" in lib.fox_last_error()
    assert decode(W=1 << 27) == -1 and b"2^30" in lib.fox_last_error()
    assert decode(most=-1) == -1 and decode(lengths=None) == -1 and decode(q=base + 4) == -2
    assert decode(W=64, n=16) == -1 and b"workspace" in lib.fox_last_error()
    assert decode(W=64, ws=None) == -1 and decode(W=64, ws=base + 8) == -2
    n = C.c_int64(-1)
    assert lib.fox_paged_decode_workspace_bytes(4, 2, 64, 256, C.byref(n)) == 0 and n.value == 0      # nobody has more than one piece
    assert lib.fox_paged_decode_workspace_bytes(4, 2, 64, 4096, C.byref(n)) == 0 and n.value > 0
    assert lib.fox_paged_decode_workspace_bytes(4, 2, 64, (1 << 30) + 1, C.byref(n)) == -1 and lib.fox_paged_decode_workspace_bytes(1 << 12, 1 << 12, 64, 64, C.byref(n)) == -1
    assert lib.fox_paged_append(None, None) == -1 and lib.fox_paged_decode(None, None) == -1 and lib.fox_page_slots(None, None) == -1 and lib.fox_page_release(None, None) == -1


def test_rotary_wrapper_refusals():
    x, f = torch.randn(2, 5, 3, 64).bfloat16(), ft.rotary_frequencies(64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.rotary(x, f)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.qk_norm_rotary(x, x, torch.ones(64), torch.ones(64), f)
    for bad in (x.float(), x[0], torch.randn(2, 5, 3, 48).bfloat16()):
        with pytest.raises(AssertionError):
            ft.rotary(bad, f)
    from forgetting_transformer.ops.rotary import _check_angles
    check = lambda f=f, p=None, inter=False, hf=False: _check_angles(x, f, p, inter, hf)
    for bad in (dict(f=ft.rotary_frequencies(24)), dict(f=ft.rotary_frequencies(128)), dict(f=f[None]), dict(f=f[:0]), dict(f=torch.ones(32, dtype=torch.long)),
                dict(f=f.clone().requires_grad_()), dict(p=torch.zeros(5)), dict(p=torch.zeros(4, dtype=torch.long)), dict(p=torch.zeros(3, 5, dtype=torch.long)),
                dict(p=torch.zeros(2, 5, 1, dtype=torch.long)), dict(p=torch.zeros(5, dtype=torch.bool)), dict(p=torch.zeros(5, dtype=torch.long), hf=True)):
        with pytest.raises(AssertionError):
            check(**bad)
    with pytest.raises(TypeError):
        check(p=1.5)
    g, p = check(f=f[:3].float(), p=torch.arange(5, dtype=torch.int32), inter=True)
    assert g.dtype == torch.float64 and p.dtype == torch.int64


def test_paged_wrapper_refusals():
    from forgetting_transformer.ops.paged import _check_pages, _check_state
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32)
    state = dict(lengths=i32(3), block_table=i32(3, 4), free_pages=i32(9), free_count=i32(1))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.page_slots(state["lengths"], i32(3), state["block_table"], state["free_pages"], state["free_count"], page_size=16, max_tokens=4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.page_release(state["lengths"], torch.zeros(3, dtype=torch.bool), state["block_table"], state["free_pages"], state["free_count"], page_size=16)
    for bad in (dict(page_size=4), dict(page_size=24), dict(lengths=torch.zeros(3)), dict(lengths=i32(3, 1))):
        with pytest.raises(AssertionError):
            _check_state(**{**state, "page_size": 16, **bad})
    k, g = torch.zeros(4, 2, 16, 64).bfloat16(), torch.zeros(4, 2, 16)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.paged_append(k[0].transpose(0, 1), k[0].transpose(0, 1), g[0].t(), k, k, g, torch.arange(16))
    with pytest.raises(RuntimeError, match="no CPU path"):
        ft.paged_forgetting_attention(torch.zeros(3, 2, 64).bfloat16(), k, k, g, state["block_table"], state["lengths"])
    for bad in ((k.float(), k.float(), g), (k, k[:3], g), (k, k.half(), g), (k, k, g.double()), (k, k, g[:, :1]), (k[:, :, :12], k[:, :, :12], g[:, :, :12]),
                (k[..., :48], k[..., :48], g)):
        with pytest.raises(AssertionError):
            _check_pages(*bad)
    for bad in (dict(page_size=10), dict(head_dim=80), dict(max_requests=5000), dict(num_pages=0), dict(dtype=torch.float32)):
        with pytest.raises(AssertionError):
            ft.PagedFgateCache(**{**dict(num_layers=1, num_heads=2, head_dim=64, num_pages=4, max_requests=2, max_length=32, device="cpu"), **bad})
