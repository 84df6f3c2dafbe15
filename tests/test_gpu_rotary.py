"""Position rotation of queries and keys, alone and behind their norms, against the formulas in 64 bits.

Tolerances.  An output of 16 bits is off by half a step of its type (eps / 2 relative; for fp16 2^-25 below its normal range) and by what 32-bit arithmetic
loses in front of that: a rotation adds two products of magnitude m = the pair's largest element with cosine and sine good to 2^-22, below 2^-20 m; the
norm adds the error of a 128-term sum of squares, below 2^-18 of the head's largest element; its gradient two such sums, below 2^-16 of the largest
term it adds.  A weight gradient is a sum of N terms, added in chains of at most 512 links: 2^-15 of the sum of magnitudes."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def turned(x, pos, freq, inter, back=False):
    """x (B, T, H, D) float64, pos (B, T): the first 2 len(freq) elements rotated, pair by pair."""
    R = 2 * len(freq)
    theta = (pos.double()[..., None] * freq)[:, :, None]
    c, s = theta.cos(), theta.sin() * (-1 if back else 1)
    y = x.clone()
    ia, ib = (slice(0, R, 2), slice(1, R, 2)) if inter else (slice(0, R // 2), slice(R // 2, R))
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ia] * s + x[..., ib] * c
    return y


def half_step(ref, dtype):
    return torch.finfo(dtype).eps / 2 * ref.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def check(name, got, ref, slack, dtype):
    bound = half_step(ref, dtype) + slack
    err = (got.double() - ref).abs()
    assert torch.isfinite(got).all(), name
    assert (err <= bound).all(), f"{name}: {(err / bound).max().item():.3f} of its bound"


def inputs(B, T, H, D, dtype, seed, head_first, positions):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(B, T, H, D, generator=g).to(dtype).cuda()
    dy = torch.randn(B, T, H, D, generator=g).to(dtype).cuda()
    pos = {"none": None, "int": 1000003, "row": torch.arange(T) + 77, "batch": torch.randint(0, 1 << 20, (B, T), generator=g),
           "start": torch.randint(-50, 1 << 30, (B, 1), generator=g)}[positions]
    full = torch.arange(T).expand(B, T) if pos is None else (pos + torch.arange(T)).expand(B, T) if isinstance(pos, int) else pos.expand(B, T)
    if head_first:
        x, dy = x.transpose(1, 2).contiguous(), dy.transpose(1, 2).contiguous()
    return x, dy, pos if not isinstance(pos, torch.Tensor) else pos.cuda(), full.cuda()


SHAPES = [  # B, T, H, D, R, interleaved, dtype, head_first, positions
    (1, 1, 1, 16, 16, False, torch.bfloat16, False, "none"), (1, 1, 1, 16, 2, True, torch.float16, True, "int"), (2, 7, 3, 32, 16, False, torch.bfloat16, True, "row"),
    (2, 7, 3, 32, 10, True, torch.bfloat16, False, "batch"), (3, 129, 5, 64, 64, False, torch.float16, False, "start"), (3, 65, 5, 64, 64, True, torch.bfloat16, True, "batch"),
    (2, 300, 12, 128, 128, False, torch.bfloat16, False, "int"), (2, 300, 12, 128, 48, False, torch.float16, True, "batch"), (1, 33, 70, 128, 96, True, torch.bfloat16, False, "none"),
    (16, 1, 16, 128, 128, False, torch.bfloat16, False, "start"), (1, 1111, 1, 16, 16, True, torch.bfloat16, False, "none"), (4, 501, 2, 64, 32, False, torch.float16, False, "row"),
    (1, 5000, 16, 64, 64, False, torch.bfloat16, True, "batch"), (1, 9, 300, 64, 16, False, torch.bfloat16, False, "row")]


@pytest.mark.parametrize("B,T,H,D,R,inter,dtype,hf,positions", SHAPES)
def test_rotary(B, T, H, D, R, inter, dtype, hf, positions):
    from forgetting_transformer import rotary, rotary_frequencies
    x, dy, pos, full = inputs(B, T, H, D, dtype, 1, hf, positions)
    freq = rotary_frequencies(R, device="cuda")
    x.requires_grad_()
    y = rotary(x, freq, positions=pos, interleaved=inter, head_first=hf)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert y.shape == x.shape and y.stride() == x.stride() and dx.shape == x.shape
    flat = lambda t: (t.transpose(1, 2) if hf else t).detach()
    for name, got, src, back in (("y", y, x, False), ("dx", dx, dy, True)):
        src = flat(src).double()
        check(name, flat(got), turned(src, full, freq, inter, back), 2.0 ** -20 * src.abs().amax(-1, keepdim=True), dtype)
        assert torch.equal(flat(got)[..., R:], src[..., R:].to(dtype))      # what is not rotated is copied
    with torch.no_grad():
        assert torch.equal(rotary(x, freq, positions=pos, interleaved=inter, head_first=hf), y)


def norm_ref(x, w, eps):
    rstd = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    return x * rstd, rstd, w


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("B,T,H,D,R,inter,dtype,hf,positions", SHAPES)
def test_qk_norm_rotary(B, T, H, D, R, inter, dtype, hf, positions, shared):
    from forgetting_transformer import qk_norm_rotary, rotary_frequencies
    q, dyq, pos, full = inputs(B, T, H, D, dtype, 2, hf, positions)
    Hk = max(1, H // 2) if H % 3 else H
    k, dyk, _, _ = inputs(B, T, Hk, D, dtype, 3, hf, positions)
    freq, eps = rotary_frequencies(R, device="cuda"), 1e-5
    g = torch.Generator().manual_seed(4)
    wq, wk = (torch.rand(D if shared else h * D, generator=g).cuda() + 0.5 for h in (H, Hk))
    leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
    yq, yk = qk_norm_rotary(q, k, wq, wk, freq, positions=pos, interleaved=inter, eps=eps, head_first=hf)
    dq, dk, dwq, dwk = torch.autograd.grad([yq, yk], leaves, [dyq, dyk])
    flat = lambda t: (t.transpose(1, 2) if hf else t).detach()
    for name, x, w, dy, y, dx, dw, h in (("q", q, wq, dyq, yq, dq, dwq, H), ("k", k, wk, dyk, yk, dk, dwk, Hk)):
        assert y.stride() == x.stride() and dx.shape == x.shape and dw.shape == w.shape and dw.dtype == w.dtype
        x64, dy64, rows = flat(x).double(), flat(dy).double(), w.detach().double().reshape(-1, D).expand(h, D)
        rstd = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
        xhat = x64 * rstd
        n = xhat * rows
        check("y" + name, flat(y), turned(n, full, freq, inter), 2.0 ** -18 * n.abs().amax(-1, keepdim=True), dtype)
        dn = turned(dy64, full, freq, inter, back=True)
        gw = dn * rows
        ref = rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True))
        largest = rstd * gw.abs().amax(-1, keepdim=True) * (1 + xhat.abs().amax(-1, keepdim=True))
        check("d" + name, flat(dx), ref, 2.0 ** -16 * largest, dtype)
        terms = dn * xhat
        total, size = terms.sum((0, 1)), terms.abs().sum((0, 1))
        if shared:
            total, size = total.sum(0), size.sum(0)
        err = (dw.double() - total.reshape(-1)).abs()
        assert (err <= 2.0 ** -15 * size.reshape(-1) + 1e-30).all(), f"dw{name}: {(err / size.reshape(-1)).max().item():.2e} of the terms' sum"


def test_gradients_against_differences():
    """The gradients of a weighted sum of the outputs, rows given in 16 bits but evaluated in 64: the formulas of the tests above against central differences."""
    g = torch.Generator().manual_seed(5)
    x, w, dy = (torch.randn(1, 2, 1, 16, generator=g, dtype=torch.float64) for _ in range(3))
    w = w[0, 0].abs() + 0.5
    pos, freq = torch.tensor([[3, 9]]), 10.0 ** -torch.arange(0, 8, dtype=torch.float64)

    def f(x, w):
        rstd = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        return (turned(x * rstd * w, pos, freq, False) * dy).sum()

    rstd = (x.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
    xhat, dn = x * rstd, turned(dy, pos, freq, False, back=True)
    dx = rstd * (dn * w - xhat * (dn * w * xhat).mean(-1, keepdim=True))
    dw = (dn * xhat).sum((0, 1))
    h = 1e-6
    for i in range(x.numel()):
        e = torch.zeros(x.numel(), dtype=torch.float64)
        e[i] = h
        e = e.view_as(x)
        assert abs((f(x + e, w) - f(x - e, w)) / (2 * h) - dx.reshape(-1)[i]) < 1e-7
    for i in range(16):
        e = torch.zeros(1, 16, dtype=torch.float64)
        e[0, i] = h
        assert abs((f(x, w + e) - f(x, w - e)) / (2 * h) - dw.reshape(-1)[i]) < 1e-7


def test_many_tokens_weight_gradient():
    """Strips of several tiles, partial sums of more rows than one launch adds, and heads beyond one workgroup's columns."""
    from forgetting_transformer import qk_norm_rotary, rotary_frequencies
    for B, T, H, D, shared in ((2, 30000, 2, 64, True), (1, 20011, 3, 32, False), (1, 2111, 40, 128, True), (1, 2111, 40, 128, False)):
        q, dyq, _, full = inputs(B, T, H, D, torch.bfloat16, 6, False, "none")
        k, dyk, _, _ = inputs(B, T, H, D, torch.bfloat16, 7, False, "none")
        freq = rotary_frequencies(D, device="cuda")
        wq, wk = (torch.rand(D if shared else H * D, device="cuda") + 0.5 for _ in range(2))
        leaves = [t.requires_grad_() for t in (q, k, wq, wk)]
        first = torch.autograd.grad(qk_norm_rotary(q, k, wq, wk, freq), leaves, [dyq, dyk])
        again = torch.autograd.grad(qk_norm_rotary(q, k, wq, wk, freq), leaves, [dyq, dyk])
        assert all(torch.equal(a, b) for a, b in zip(first, again))           # a fixed order of additions
        for x, dy, dw in ((q, dyq, first[2]), (k, dyk, first[3])):
            x64 = x.detach().double()
            terms = turned(dy.double(), full, freq, False, back=True) * x64 * (x64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
            total, size = terms.sum((0, 1)), terms.abs().sum((0, 1))
            if shared:
                total, size = total.sum(0), size.sum(0)
            assert ((dw.double() - total.reshape(-1)).abs() <= 2.0 ** -15 * size.reshape(-1)).all()


def test_far_positions():
    """Angles at positions that 32 bits cannot hold: whole turns are taken off in 64 bits."""
    from forgetting_transformer import rotary, rotary_frequencies
    x = torch.randn(1, 4, 2, 64, device="cuda").bfloat16()
    freq = rotary_frequencies(64, device="cuda")
    for p in (2 ** 24 + 1, 2 ** 31 - 3, -(2 ** 31), 2 ** 33 + 12345):
        pos = p + torch.arange(4, device="cuda")
        ref = turned(x.double(), pos[None], freq, False)
        slack = (2.0 ** -20 + abs(p) * 2.0 ** -50) * x.double().abs().amax(-1, keepdim=True)   # (an angle of 64 bits is off by 2^-53 of itself, here and there)
        check("y", rotary(x, freq, positions=pos), ref, slack, torch.bfloat16)
        assert torch.equal(rotary(x, freq, positions=p), rotary(x, freq, positions=pos))


def test_infinities_stay_in_their_pair():
    from forgetting_transformer import rotary, rotary_frequencies
    for inter, R in ((False, 32), (True, 32), (True, 6)):
        x = torch.randn(1, 3, 2, 64, device="cuda").bfloat16()
        y = rotary(x, rotary_frequencies(R, device="cuda"), interleaved=inter, positions=5)
        z = x.clone()
        z[..., R:] = float("inf")
        z[0, 0, 0, R] = float("nan")
        got = rotary(z, rotary_frequencies(R, device="cuda"), interleaved=inter, positions=5)
        assert torch.equal(got[..., :R], y[..., :R]) and torch.equal(got[..., R:].nan_to_num(7.0, 9.0), z[..., R:].nan_to_num(7.0, 9.0))
        z = x.clone()
        z[0, 1, 1, 3] = float("inf")
        pair = (2, 3) if inter else (3, 3 + R // 2)
        rest = [d for d in range(64) if d not in pair]
        got = rotary(z, rotary_frequencies(R, device="cuda"), interleaved=inter, positions=5)
        assert torch.equal(got[0, 1, 1, rest], y[0, 1, 1, rest]) and torch.equal(got[0, 0], y[0, 0])


def test_layouts_types_and_converted_arguments():
    """Views with gaps, unaligned ones, weights and frequencies of other types, int32 positions: as the plain call."""
    from forgetting_transformer import qk_norm_rotary, rotary, rotary_frequencies
    B, T, H, D = 2, 50, 3, 64
    big = torch.randn(B, T, 2 * H * D + 8, device="cuda").bfloat16()
    freq = rotary_frequencies(D, device="cuda")
    x = big[..., 8:8 + H * D].view(B, T, H, D)
    off = big[..., 3:3 + H * D].view(B, T, H, D)                  # 2-byte aligned only
    for t in (x, off, x.transpose(1, 2).contiguous().transpose(1, 2), x.expand(B, T, H, D)):
        assert torch.equal(rotary(t, freq), rotary(t.contiguous(), freq))
        t = t.detach().requires_grad_()
        y = rotary(t, freq)
        (dx,) = torch.autograd.grad(y, t, torch.ones_like(y))
        (ref,) = torch.autograd.grad(rotary(u := t.detach().contiguous().requires_grad_(), freq), u, torch.ones(B, T, H, D, device="cuda").bfloat16())
        assert torch.equal(dx, ref)
    assert torch.equal(rotary(x, freq, positions=torch.arange(T, dtype=torch.int32)), rotary(x, freq))
    odd = torch.randn(1 + D, device="cuda").bfloat16()[1:].view(1, 1, 1, D)        # contiguous, but not where a 16-byte vector may start
    y = rotary(odd.requires_grad_(), freq, positions=3)
    assert torch.equal(y, rotary(odd.detach().clone(), freq, positions=3))
    assert torch.equal(torch.autograd.grad(y, odd, odd.detach())[0], rotary(odd.detach().clone(), freq, positions=-3))
    assert torch.equal(rotary(x[:1].expand(B, T, H, D), freq), rotary(x[:1].repeat(B, 1, 1, 1), freq))
    single = freq.float()
    assert torch.equal(rotary(x, single), rotary(x, single.double()))
    wq, wk = torch.rand(H * D, device="cuda"), torch.rand(H * D, device="cuda")
    k = x.flip(0).contiguous()
    want = qk_norm_rotary(x, k, wq.bfloat16().float(), wk.bfloat16().float(), freq)
    got = qk_norm_rotary(x, k, wq.bfloat16().requires_grad_(), wk.bfloat16(), freq)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    w = wq.bfloat16().requires_grad_()
    (dw,) = torch.autograd.grad(qk_norm_rotary(x, k, w, wk, freq)[0].float().sum(), w)
    assert dw.dtype == torch.bfloat16
    odd = torch.rand(H * D + 1, device="cuda")[1:]                # 4-byte aligned weights
    assert torch.equal(qk_norm_rotary(x, k, odd, wk, freq)[0], qk_norm_rotary(x, k, odd.clone(), wk, freq)[0])


def test_views_beyond_32_bits():
    """Tokens whose rows lie further apart than 2^31 elements in all, forward and back, as packed ones."""
    from forgetting_transformer import qk_norm_rotary, rotary, rotary_frequencies
    T, H, D, gap = 600, 2, 64, 1 << 22
    freq = rotary_frequencies(D, device="cuda")
    mem = torch.empty(T * gap, dtype=torch.bfloat16, device="cuda")
    far = [mem.as_strided((1, T, H, D), (T * gap, gap, D, 1), i * H * D) for i in range(4)]
    near = [torch.randn(1, T, H, D, device="cuda").bfloat16() for _ in far]
    for dst, src in zip(far, near):
        dst.copy_(src)
    assert torch.equal(rotary(far[0], freq), rotary(near[0], freq))
    results = []
    for q, k, dyq, dyk in (far, near):
        leaves = [t.detach().requires_grad_() for t in (q, k)] + [torch.linspace(0.5, 1.5, D, device="cuda").requires_grad_() for _ in range(2)]
        y = qk_norm_rotary(*leaves, freq)
        results.append([*y, *torch.autograd.grad(y, leaves, [dyq, dyk])])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_many_tokens_as_their_parts():
    """Rows do not depend on the call they are in: 2^24 and some tokens at once and in parts from their positions on."""
    from forgetting_transformer import qk_norm_rotary, rotary, rotary_frequencies
    T, D, cut = (1 << 24) + 77, 16, 1 << 19
    freq, w = rotary_frequencies(D, device="cuda"), torch.linspace(0.5, 1.5, D, device="cuda")
    x = torch.randn(1, T, 1, D, device="cuda").bfloat16()
    k = x.flip(1)
    y, (yq, yk) = rotary(x, freq), qk_norm_rotary(x, k, w, w, freq)
    leaf = x.detach().requires_grad_()
    (dx,) = torch.autograd.grad(qk_norm_rotary(leaf, k, w, w, freq)[0], leaf, k)
    for at in (0, 5 * cut + 3, T - cut):
        part = slice(at, at + cut)
        assert torch.equal(y[:, part], rotary(x[:, part], freq, positions=at))
        leaf = x[:, part].detach().requires_grad_()
        pq, pk = qk_norm_rotary(leaf, k[:, part], w, w, freq, positions=at)
        assert torch.equal(yq[:, part], pq) and torch.equal(yk[:, part], pk)
        assert torch.equal(dx[:, part], torch.autograd.grad(pq, leaf, k[:, part])[0])


def test_unused_outputs_second_derivatives_and_empty_calls():
    from forgetting_transformer import qk_norm_rotary, rotary, rotary_frequencies
    freq = rotary_frequencies(32, device="cuda")
    x = torch.randn(2, 9, 4, 32, device="cuda").half().requires_grad_()
    k = torch.randn(2, 9, 4, 32, device="cuda").half().requires_grad_()
    w = torch.ones(32, device="cuda", requires_grad=True)
    yq, _ = qk_norm_rotary(x, k, w, torch.ones(32, device="cuda"), freq)
    dq, dk = torch.autograd.grad(yq.float().sum(), [x, k])
    assert dq.abs().max() > 0 and dk.abs().max() == 0
    v = torch.randn_like(x).requires_grad_()
    (dx,) = torch.autograd.grad(rotary(x, freq, positions=3), x, v, create_graph=True)
    (dv,) = torch.autograd.grad(dx, v, x.detach())                # the gradient of the turned-back v is the turned x
    assert torch.equal(dv, rotary(x.detach(), freq, positions=3))
    yq, _ = qk_norm_rotary(x, k, w, w, freq)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(yq.float().sum(), x, create_graph=True)
    for shape in ((0, 5, 2, 32), (2, 0, 2, 32)):
        e = torch.empty(shape, device="cuda", dtype=torch.half, requires_grad=True)
        assert rotary(e, freq).shape == shape
        yq, yk = qk_norm_rotary(e, e, w, w, freq)
        de, dw = torch.autograd.grad([yq, yk], [e, w], [torch.empty_like(yq), torch.empty_like(yk)])
        assert de.shape == shape and dw.abs().max() == 0
    with pytest.raises(AssertionError):
        qk_norm_rotary(x, k, torch.ones(32, device="cuda"), torch.ones(128, device="cuda"), freq)
    with pytest.raises(AssertionError):
        qk_norm_rotary(x, k[:, :4], w, w, freq)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: rotary(t, freq))(x.detach()[None])


def test_streams_and_graph_replay():
    """On another stream, and forward and backward captured and replayed on new contents beside eager work, bit for bit."""
    from forgetting_transformer import qk_norm_rotary, rotary_frequencies
    freq = rotary_frequencies(64, device="cuda")
    pos = torch.arange(200, device="cuda")
    sets = [[torch.randn(2, 200, 4, 64, device="cuda").bfloat16() for _ in range(4)] + [torch.rand(256, device="cuda"), torch.rand(256, device="cuda")] for _ in range(3)]

    def step(q, k, dyq, dyk, wq, wk):
        leaves = [t.detach().requires_grad_() for t in (q, k, wq, wk)]
        y = qk_norm_rotary(*leaves, freq, positions=pos)
        return [*(t.detach() for t in y), *torch.autograd.grad(y, leaves, [dyq, dyk])]

    eager = [[t.clone() for t in step(*s)] for s in sets]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(*sets[1])
        static = [t.clone() for t in sets[0]]
        step(*static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(other, eager[1]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(*static)
    for _ in range(2):
        for s, want in zip(sets, eager):
            for dst, src in zip(static, s):
                dst.copy_(src)
            graph.replay()
            torch.cuda.synchronize()
            torch.randn(1 << 20, device="cuda").sum().item()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_c_entry():
    """One side alone through the C entry, on strided views, from a position on; forward and back."""
    import ctypes as C
    from forgetting_transformer import rotary, rotary_frequencies
    from forgetting_transformer.ops import _lib
    lib = _lib.load()
    x = torch.randn(2, 30, 5, 64, device="cuda").bfloat16()
    mem = torch.zeros(2, 5, 40, 72, dtype=torch.bfloat16, device="cuda")
    y = mem[:, :, 3:33, :64].transpose(1, 2)
    freq = rotary_frequencies(32, device="cuda")
    view = lambda t: _lib.View(t.data_ptr(), t.stride(0), t.stride(2), t.stride(1))
    none = _lib.View(None, 0, 0, 0)

    def args(a, b, dx):
        side = _lib.RotarySide(5, a, b, dx, None)
        return _lib.RotaryArgs(1, 2, 30, 64, 0, 32, 0, (_lib.RotarySide * 2)(side, _lib.RotarySide()), 0, 0.0, freq.data_ptr(), None, 0, 0, 11, None, None)

    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(lib.fox_rotary_fwd(C.byref(args(view(x), view(y), none)), stream), "fox_rotary_fwd")
    assert torch.equal(y, rotary(x, freq, positions=11))
    back = torch.empty_like(x)
    _lib.check(lib.fox_rotary_bwd(C.byref(args(none, view(y), view(back))), stream), "fox_rotary_bwd")
    assert torch.equal(back, rotary(y.contiguous(), freq, positions=-torch.arange(11, 41, device="cuda")))
    assert mem.abs().sum() == y.abs().sum()                              # nothing beside the view


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("sides", [1, 2])
@pytest.mark.parametrize("B,T,H,D", [(2, 30, 5, 64), (1, 1, 1, 16), (1, 700, 40, 128)])
def test_c_entry_norm_gradients_stay_in_their_buffers(B, T, H, D, sides, shared):
    """Norm and rotation through the C entry with one side and with two: right gradients, and nothing behind dweight and the workspace."""
    import ctypes as C
    from forgetting_transformer import rotary_frequencies
    from forgetting_transformer.ops import _lib
    lib = _lib.load()
    gen = torch.Generator(device="cuda").manual_seed(8)
    x, dy = ([torch.randn(B, T, H, D, generator=gen, device="cuda").bfloat16() for _ in range(sides)] for _ in range(2))
    w = [torch.rand(1 if shared else H, D, generator=gen, device="cuda") + 0.5 for _ in range(sides)]
    y, dx = ([torch.empty_like(t) for t in x] for _ in range(2))
    freq, eps, n = rotary_frequencies(16, device="cuda"), 1e-5, C.c_int64()
    _lib.check(lib.fox_rotary_workspace_bytes(B * T, sides * H, D, shared, C.byref(n)), "fox_rotary_workspace_bytes")
    used, guard = sides * w[0].numel(), 4 * D
    dw = torch.full((used + guard,), 7.0, device="cuda")
    ws = torch.full((n.value // 4 + guard,), 7.0, device="cuda")
    view = lambda t: _lib.View(t.data_ptr(), t.stride(0), t.stride(2), t.stride(1))
    side = lambda i: _lib.RotarySide(H, view(x[i]), view(y[i] if forward else dy[i]), view(dx[i]), w[i].data_ptr()) if i < sides else _lib.RotarySide()
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    for forward in (True, False):
        args = _lib.RotaryArgs(sides, B, T, D, 0, 16, 0, (_lib.RotarySide * 2)(side(0), side(1)), 0 if shared else D, eps, freq.data_ptr(), None, 0, 0, 11,
                               dw.data_ptr(), ws.data_ptr())
        _lib.check((lib.fox_rotary_fwd if forward else lib.fox_rotary_bwd)(C.byref(args), stream), "fox_rotary")
    assert (dw[used:] == 7.0).all() and (ws[n.value // 4:] == 7.0).all()
    full = (11 + torch.arange(T, device="cuda")).expand(B, T)
    for i in range(sides):
        x64 = x[i].double()
        rstd = (x64.square().mean(-1, keepdim=True) + eps).rsqrt()
        xhat, dn = x64 * rstd, turned(dy[i].double(), full, freq, False, back=True)
        out, gw = xhat * w[i].double(), dn * w[i].double()
        check("y", y[i], turned(out, full, freq, False), 2.0 ** -18 * out.abs().amax(-1, keepdim=True), torch.bfloat16)
        largest = rstd * gw.abs().amax(-1, keepdim=True) * (1 + xhat.abs().amax(-1, keepdim=True))
        check("dx", dx[i], rstd * (gw - xhat * (gw * xhat).mean(-1, keepdim=True)), 2.0 ** -16 * largest, torch.bfloat16)
        terms = dn * xhat
        total, size = terms.sum((0, 1)), terms.abs().sum((0, 1))
        if shared:
            total, size = total.sum(0), size.sum(0)
        got = dw[:used].view(sides, -1)[i].double()
        assert ((got - total.reshape(-1)).abs() <= 2.0 ** -15 * size.reshape(-1) + 1e-30).all()


@pytest.mark.parametrize("inter", [False, True])
def test_small_angles_keep_their_digits(inter):
    """Unit vectors turn into the cosine and the sine themselves: off by the output's rounding, 2^-22 of their own magnitude (not of the pair's: a low frequency's first
    positions have sines of 1e-4) and what 64-bit arithmetic leaves of the angle, some 2^-51 of it."""
    from forgetting_transformer import rotary, rotary_frequencies
    T, D, dtype = 3000, 128, torch.float16
    freq = rotary_frequencies(D, device="cuda")
    x = torch.zeros(1, T, 1, D, device="cuda", dtype=dtype)
    x[..., slice(0, D, 2) if inter else slice(0, D // 2)] = 1.0
    for first in (0, -700, 1 << 20):
        y = rotary(x, freq, positions=first, interleaved=inter)[0, :, 0].double()
        theta = (first + torch.arange(T, device="cuda")).double()[:, None] * freq
        for got, ref in zip((y[:, 0::2], y[:, 1::2]) if inter else (y[:, :D // 2], y[:, D // 2:]), (theta.cos(), theta.sin())):
            bound = half_step(ref, dtype) * (1 + 2.0 ** -10) + 2.0 ** -22 * ref.abs() + 2.0 ** -50 * theta.abs()
            err = (got - ref).abs()
            assert (err <= bound).all(), f"{(err / bound).max().item():.3f} of its bound at {first}"


def test_norm_of_tiny_rows():
    """Without eps the norm of a row does not depend on its magnitude, also where the mean square lies below the normal range of fp32 (2^-132 here, exact)."""
    from forgetting_transformer import qk_norm_rotary, rms_norm, rotary_frequencies
    D = 64
    sign = torch.where(torch.rand(1, 9, 2, D, device="cuda") < 0.5, -1.0, 1.0).bfloat16()
    freq = rotary_frequencies(D, device="cuda") * 0
    w = torch.rand(2 * D, device="cuda") + 0.5
    for scale in (1.0, 2.0 ** -60, 2.0 ** -66):
        leaves = [(sign * scale).requires_grad_(), sign.clone().requires_grad_(), w.clone().requires_grad_(), w.clone().requires_grad_()]
        yq, yk = qk_norm_rotary(*leaves, freq, eps=0.0)
        assert torch.equal(yq, (sign * w.view(2, D)).bfloat16()) and torch.equal(yq, yk)
        g = torch.autograd.grad([yq, yk], leaves, [sign, sign])
        assert torch.equal(g[2], g[3])
        assert torch.equal(g[0].double() * scale, g[1].double())


def test_too_many_elements():
    """Refused as an argument, before anything is allocated for the result."""
    from forgetting_transformer import qk_norm_rotary, rotary, rotary_frequencies
    freq, w = rotary_frequencies(128, device="cuda"), torch.ones(128, device="cuda")
    x = torch.zeros(1, 1, 1, 128, device="cuda").bfloat16()
    before = torch.cuda.max_memory_allocated()
    for wide, part in ((x.expand(1 << 14, 1 << 12, 3, 128), x.expand(1 << 14, 1 << 12, 2, 128)), (x.expand(1 << 15, 1 << 12, 2, 128), x.expand(1 << 15, 1 << 12, 1, 128))):
        with pytest.raises(AssertionError, match="elements"):
            rotary(wide, freq)
        with pytest.raises(AssertionError, match="elements"):
            qk_norm_rotary(part, part if wide.shape[2] == 3 else wide, w, w, freq)
    assert torch.cuda.max_memory_allocated() == before


def test_weight_gradient_in_two_launches():
    """Heads of several workgroups that share weights: more partial rows than one launch adds (512 and some), here 513 and the two groups' sums behind them."""
    import ctypes as C
    from forgetting_transformer import qk_norm_rotary, rotary_frequencies
    from forgetting_transformer.ops import _lib
    B, T, H, D = 1, 15000, 40, 128
    n = C.c_int64()
    _lib.check(_lib.load().fox_rotary_workspace_bytes(B * T, 2 * H, D, 1, C.byref(n)), "fox_rotary_workspace_bytes")
    assert n.value > 512 * 2 * D * 4
    q, dyq, _, full = inputs(B, T, H, D, torch.bfloat16, 9, False, "none")
    k, dyk, _, _ = inputs(B, T, H, D, torch.bfloat16, 10, False, "none")
    freq = rotary_frequencies(D, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, *(torch.rand(D, device="cuda") + 0.5 for _ in range(2)))]
    first = torch.autograd.grad(qk_norm_rotary(*leaves, freq), leaves, [dyq, dyk])
    again = torch.autograd.grad(qk_norm_rotary(*leaves, freq), leaves, [dyq, dyk])
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    for x, dy, dw in ((q, dyq, first[2]), (k, dyk, first[3])):
        x64 = x.detach().double()
        terms = turned(dy.double(), full, freq, False, back=True) * x64 * (x64.square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        assert ((dw.double() - terms.sum((0, 1, 2))).abs() <= 2.0 ** -15 * terms.abs().sum((0, 1, 2))).all()
