"""Attention over packed sequences: forward and gradients against the formulas in 64 bits, and against differences of the forward's formula.

Tolerances, with u half a step of the 16-bit type (``torch.finfo(t).eps / 2``), element by element:
  o    u |o| for its own rounding, u p|v| for that of the probabilities in the product with v
  dv   u |dv| + u p^T|do|
  dk   u |dk| + u scale |ds|^T|q|, and scale e_ds^T|q| for the 32-bit error e_ds of ds before it is rounded (as under dg: with a single key ds is the difference of
       two equal numbers, zero in the formula and that error in any arithmetic)
  dq   u |dq| + u scale |ds||k| + scale e_ds|k|, and what o.do is off by (delta), scale e (p|k|) with e the bound of o times |do|
  dg   32-bit arithmetic: a dot product of up to 128 terms is off by 2^-17 of the sum of their magnitudes, so a score by 2^-17 scale |q||k|, the bias by 2^-20 of itself (a difference
       of sums in 64 bits, rounded a few times on the way), a probability by as much of itself, dP by 2^-17 |do||v|; a gate's gradient adds
       columns of dS from its key on.  That is the worst case; errors of either sign add up to far less, so the norm of the error is held to 2^-16 of the gradient's too.
fp16 has no steps below 2^-24, so an entry of p or ds may be off by 2^-25 whatever its size (the largest p of a row is at least 1 before it is divided by the row's sum): n 2^-25 of the largest
value that it multiplies; and half of such a step, 2^-25, is what an output below 2^-14 may lose by its own rounding (a single key: dk is the 32-bit error of ds times q, some 4e-8, and
the nearest fp16 are 0 and 6e-8).  To all of them comes the scores' own error, 2^-14 of the same sums (scores up to 8 in size)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def inputs(new, front, H, Hk, D, dtype, seed=0, lead=0, pad=0, gate=3.0, layout="rows", scale=1.0):
    """q, k, v, log gates, dout and the ends; `lead` and `pad` places that belong to nobody hold NaN."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    T, N = lead + sum(new) + pad, lead + sum(new) + sum(front) + pad
    nobody = float("nan")

    def rnd(tokens, heads):
        if layout == "heads":        # (heads, tokens, D) memory
            x = (torch.randn(heads, tokens, D, generator=g, device="cuda") * scale).to(dtype).transpose(0, 1)
        elif layout == "wide":       # a part of a wider row
            x = (torch.randn(tokens, heads + 2, D, generator=g, device="cuda") * scale).to(dtype)[:, 1:-1]
        else:
            x = (torch.randn(tokens, heads, D, generator=g, device="cuda") * scale).to(dtype)
        x[:lead] = nobody
        x[tokens - pad:] = nobody
        return x
    q, k, v, do = rnd(T, H), rnd(N, Hk), rnd(N, Hk), rnd(T, H)
    f = torch.nn.functional.logsigmoid(torch.randn(N, H, generator=g, device="cuda") + gate)
    f[:lead], f[N - pad:] = nobody, nobody
    ends = lambda n: torch.tensor([lead] + n, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)
    return q, k, v, f, do, ends(new), ends([a + b for a, b in zip(new, front)])


def sequence(q, k, v, f, do, scale):
    """One sequence in 64 bits, all heads: o and the gradients by their formulas, and the bounds of the module's docstring (without u)."""
    H, group = q.shape[1], q.shape[1] // k.shape[1]
    q, do, f = (x.double().transpose(0, 1) for x in (q, do, f))
    k, v = (x.double().transpose(0, 1).repeat_interleave(group, 0) for x in (k, v))
    m, n = q.shape[1], k.shape[1]
    c = f.clamp(min=-1e6).cumsum(-1)
    at = torch.arange(m, device="cuda") + n - m
    see = torch.arange(n, device="cuda")[None] <= at[:, None]
    bias = c[:, at.clamp(min=0)][..., None] - c[:, None]
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()) * scale + bias
    s = s.masked_fill(~see, -math.inf)
    p = torch.nan_to_num(torch.softmax(s, -1))
    mul = lambda a, b: torch.matmul(a, b.contiguous())
    o = mul(p, v)
    dp = mul(do, v.transpose(-1, -2))
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk, dv = mul(ds, k) * scale, mul(ds.transpose(-1, -2), q) * scale, mul(p.transpose(-1, -2), do)
    back = lambda x: x.flip(-1).cumsum(-1).flip(-1)
    dg = back(-ds.sum(-2))
    dg[:, 0] = 0
    a = lambda x: x.abs()
    # (scores for the errors that a probability has relative to itself)
    rel = 2.0 ** -17 * abs(scale) * mul(a(q), a(k).transpose(-1, -2)) + 2.0 ** -20 * torch.where(see, bias.abs(), 0.0)
    e_dp = 2.0 ** -17 * mul(a(do), a(v).transpose(-1, -2))
    row = (p * (e_dp + rel * a(dp))).sum(-1, keepdim=True)
    e_ds = p * (e_dp + rel * a(dp - delta) + row)
    join = lambda x: x.unflatten(0, (H // group, group)).sum(1)      # over the heads of a group
    e_o = mul(p, a(v)) + a(o)
    e_dq = abs(scale) * (mul(a(ds), a(k)) + (e_o * a(do)).sum(-1, keepdim=True) * mul(p, a(k))) + a(dq)
    e_dk = abs(scale) * join(mul(a(ds).transpose(-1, -2), a(q)))
    n_dq, n_dk = abs(scale) * mul(e_ds, a(k)), abs(scale) * join(mul(e_ds.transpose(-1, -2), a(q)))
    e_dv = join(mul(p.transpose(-1, -2), a(do)))
    dk, dv = join(dk), join(dv)
    t = lambda x: x.transpose(0, 1)
    tiny = 2.0 ** -25 * max(m, n) * group                            # of the largest factor: fp16 only
    small = [x + 2.0 ** -25 for x in (tiny * v.abs().max(), tiny * abs(scale) * k.abs().max(), tiny * abs(scale) * q.abs().max(), tiny * do.abs().max())]
    noise = [0.0, t(n_dq), t(n_dk), 0.0]                             # not in steps of the type
    return [t(x) for x in (o, dq, dk, dv, dg)], [t(x) for x in (e_o, e_dq, e_dk + a(dk), e_dv + a(dv))], t(back(e_ds.sum(-2))), small, noise


def check(x, cu_q, cu_k, scale, got, dtype):
    q, k, v, f, do = x
    u = torch.finfo(dtype).eps / 2
    names = ("o", "dq", "dk", "dv", "dg")
    ends_q, ends_k = cu_q.tolist(), cu_k.tolist()
    wrong, size = 0.0, 0.0
    for b in range(len(ends_q) - 1):
        rq, rk = slice(ends_q[b], ends_q[b + 1]), slice(ends_k[b], ends_k[b + 1])
        if rq.start == rq.stop and rk.start == rk.stop:
            continue
        if rq.start == rq.stop or rk.start == rk.stop:      # keys without queries, queries without keys
            for y, r in zip(got, (rq, rq, rk, rk, rk)):
                assert not y[r].any()
            continue
        want, bound, e_dg, small, noise = sequence(q[rq], k[rk], v[rk], f[rk], do[rq], scale)
        for name, y, w, e, r, tiny, own in zip(names, got, want, bound, (rq, rq, rk, rk), small, noise):
            err, top = (y[r].double() - w).abs(), (u + 2.0 ** -14) * e + own + (tiny if dtype == torch.float16 else 0.0) + 1e-30
            assert torch.isfinite(y[r]).all(), name
            assert (err <= top).all(), f"{name} of sequence {b}: {(err / top).max().item():.3f} of its bound"
        if len(got) == 5:
            err = (got[4][rk].double() - want[4]).abs()
            top = e_dg + 2.0 ** -24 * want[4].abs() + 1e-30
            assert (err <= top).all(), f"dg of sequence {b}: {(err / top).max().item():.3f} of its bound"
            wrong, size = wrong + err.square().sum().item(), size + want[4].square().sum().item()
    for y, ends in zip(got, (ends_q, ends_q, ends_k, ends_k, ends_k)):
        assert not y[:ends[0]].any() and not y[ends[-1]:].any()
    return wrong ** 0.5, size ** 0.5


CASES = [  # new tokens, tokens in front, H, Hk, D, dtype, more
    ([1], [0], 1, 1, 16, torch.bfloat16, {}),
    ([1, 1, 1], [0, 5, 64], 3, 1, 32, torch.float16, dict(pad=1)),
    ([2, 0, 129, 64, 63], [0, 0, 0, 0, 0], 2, 2, 64, torch.bfloat16, dict(pad=200, lead=3)),
    ([128, 127, 1, 300], [0, 1, 700, 0], 4, 2, 128, torch.float16, dict(layout="heads")),
    ([640, 31], [0, 0], 8, 1, 128, torch.bfloat16, dict(layout="wide")),
    ([5, 1000, 17], [11, 24, 333], 6, 2, 64, torch.bfloat16, dict(lead=130, pad=5)),
    ([700], [0], 12, 12, 32, torch.bfloat16, dict(gate=-2.0)),
    ([400, 260], [0, 100], 16, 4, 16, torch.float16, dict(layout="heads", pad=129)),
    ([1500], [0], 8, 8, 128, torch.bfloat16, dict(gate=6.0)),
    ([130, 5], [900, 1300], 16, 8, 128, torch.bfloat16, {}),
    ([3] * 150, [0] * 150, 5, 5, 64, torch.bfloat16, dict(pad=7)),
    ([60, 200], [-20, -200], 4, 2, 64, torch.bfloat16, {}),           # more queries than keys: the first see none; none at all
    ([100, 0, 300], [-100, 50, -299], 3, 3, 128, torch.float16, {}),
    # walks that are cut: rows of the one head, heads of a group, both; a few queries far into their keys; queries without keys at the top
    ([1800, 40, 3], [0, 0, 0], 1, 1, 64, torch.bfloat16, dict(lead=5)),
    ([900, 12], [0, 0], 8, 1, 64, torch.float16, dict(pad=3)),
    ([1300, 5], [0, 50], 2, 1, 128, torch.bfloat16, {}),
    ([2, 130], [6000, 10], 2, 2, 32, torch.bfloat16, {}),
    ([1], [9000], 16, 4, 16, torch.float16, {}),
    ([1500, 20], [-700, 0], 1, 1, 128, torch.bfloat16, {}),
    # many sequences, long ones among them
    ([3] * 130 + [900, 2, 700], [0] * 131 + [5, 300], 2, 1, 64, torch.bfloat16, dict(pad=4)),
    ([1, 0, 2] * 400 + [600], [2, 0, 0] * 400 + [0], 2, 2, 16, torch.float16, dict(lead=2)),
    # gates that need their sums in two parts at the diagonal, everywhere and in some tiles
    ([600, 300], [0, 100], 4, 2, 128, torch.bfloat16, dict(gate=-2.0)),
    ([900], [50], 3, 1, 64, torch.bfloat16, dict(gate=-3.0)),
    ([1000, 400], [0, 70], 4, 4, 64, torch.bfloat16, dict(gate=2.2)),
    ([500, 300], [0, 0], 2, 1, 128, torch.float16, dict(gate=2.2)),
]


@pytest.mark.parametrize("new,front,H,Hk,D,dtype,more", CASES)
def test_packed(new, front, H, Hk, D, dtype, more):
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs(new, front, H, Hk, D, dtype, seed=len(new) + D, **more)
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    same = not any(front)
    out = forgetting_attention_packed(*leaves, cu_q, None if same else cu_k)
    assert out.dtype == dtype and out.shape == x[0].shape
    got = [out.detach(), *torch.autograd.grad(out, leaves, x[4])]
    for y, t in zip(got[1:], x):
        assert y.shape == t.shape and y.dtype == t.dtype
    wrong, size = check(x, cu_q, cu_k, D ** -0.5, got, dtype)
    assert wrong <= 2.0 ** -16 * size
    with torch.no_grad():
        assert torch.equal(forgetting_attention_packed(*x[:4], cu_q, None if same else cu_k), out)
    again = forgetting_attention_packed(*leaves, cu_q, None if same else cu_k)
    for a, b in zip(got[1:], torch.autograd.grad(again, leaves, x[4])):
        assert torch.equal(a, b)


@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 0.3])
def test_packed_scales(scale):
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([300, 77, 500], [0, 40, 0], 4, 2, 64, torch.bfloat16, seed=3)
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = forgetting_attention_packed(*leaves, cu_q, cu_k, sm_scale=scale)
    check(x, cu_q, cu_k, scale, [out.detach(), *torch.autograd.grad(out, leaves, x[4])], torch.bfloat16)


@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
def test_packed_closed_gates(D, dtype):
    """Gates of -inf and of the type's lowest value close: nothing in front of them is seen from behind."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([400, 90, 33], [0, 0, 200], 4, 2, D, dtype, seed=5)
    f = x[3]
    f[50], f[200], f[201], f[350, 1] = -math.inf, torch.finfo(torch.float32).min, -math.inf, -math.inf
    f[400], f[495:500] = -math.inf, -math.inf                      # the first gate of a sequence, several in a row
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = forgetting_attention_packed(*leaves, cu_q, cu_k)
    check(x, cu_q, cu_k, D ** -0.5, [out.detach(), *torch.autograd.grad(out, leaves, x[4])], dtype)


@pytest.mark.parametrize("D,dtype", [(16, torch.bfloat16), (64, torch.float16), (128, torch.bfloat16)])
def test_packed_dq_of_few_keys(D, dtype):
    """Rows that see up to 32 keys: dq within its own rounding and that of ds, without the part of the module's bound that comes from the rounded o."""
    from forgetting_transformer import forgetting_attention_packed
    new = [2, 1, 3, 32, 7, 2, 20, 100, 2, 31]
    *x, cu_q, cu_k = inputs(new, [0] * len(new), 4, 2, D, dtype, seed=31)
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    got = torch.autograd.grad(forgetting_attention_packed(*leaves, cu_q), leaves, x[4])[0]
    u, scale, ends = torch.finfo(dtype).eps / 2, D ** -0.5, cu_q.tolist()
    for at, n in zip(ends, new):
        r = slice(at, at + min(n, 32))
        q, k, v, f, do = (t[r] for t in x)
        want, _, _, small, noise = sequence(q, k, v, f, do, scale)
        q, do, k, v = (t.double().transpose(0, 1).repeat_interleave(4 // t.shape[1], 0) for t in (q, do, k, v))
        c = f.double().cumsum(0).t()
        s = (torch.matmul(q, k.transpose(-1, -2)) * scale + c[..., None] - c[:, None]).masked_fill(~torch.ones(len(c[0]), len(c[0]), dtype=torch.bool, device="cuda").tril(), -math.inf)
        p, dp = torch.softmax(s, -1), torch.matmul(do, v.transpose(-1, -2))
        ds = p * (dp - (p * dp).sum(-1, keepdim=True))
        bound = (u + 2.0 ** -14) * (want[1].abs() + scale * torch.matmul(ds.abs(), k.abs()).transpose(0, 1)) + noise[1] + (small[1] if dtype == torch.float16 else 0.0) + 1e-30
        err = (got[r].double() - want[1]).abs()
        assert (err <= bound).all(), (n, (err / bound).max().item())


def test_packed_gradients_against_differences():
    """The kernels' gradients along directions against central differences of the forward's formula in 64 bits."""
    from forgetting_transformer import forgetting_attention_packed
    new, front, H, Hk, D = [70, 130], [30, 0], 4, 2, 32
    *x, cu_q, cu_k = inputs(new, front, H, Hk, D, torch.bfloat16, seed=8)
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = forgetting_attention_packed(*leaves, cu_q, cu_k)
    grads = torch.autograd.grad(out, leaves, x[4])
    ends_q, ends_k = cu_q.tolist(), cu_k.tolist()
    u = 2.0 ** -8

    def loss(y):
        return sum((sequence(y[0][ends_q[b]:ends_q[b + 1]], *(t[ends_k[b]:ends_k[b + 1]] for t in y[1:4]), x[4][ends_q[b]:ends_q[b + 1]], D ** -0.5)[0][0] *
                    x[4][ends_q[b]:ends_q[b + 1]].double()).sum().item() for b in range(2))

    gen = torch.Generator(device="cuda").manual_seed(9)
    for i in range(4):
        w = torch.randn(x[i].shape, generator=gen, device="cuda", dtype=torch.float64)
        h = 1e-5
        y = [t.double() for t in x[:4]]
        ends = []
        for sign in (1, -1):
            z = list(y)
            z[i] = y[i] + sign * h * w
            ends.append(loss(z))
        want, got = (ends[0] - ends[1]) / (2 * h), (grads[i].double() * w).sum().item()
        # rounded entries are off by about 2 u of themselves, in either direction: six times the root of the sum of their squares
        room = 6 * 2 * u * (grads[i].double() * w).square().sum().sqrt().item() if i < 3 else 1e-4 * (grads[i].double() * w).abs().sum().item()
        assert abs(want - got) <= room + 1e-5 * abs(want), (i, want, got, room)


def test_packed_equals_the_dense_operator():
    """Sequences of one length are a batch: the two operators share their tiles and differ by roundings."""
    from forgetting_transformer import forgetting_attention, forgetting_attention_packed
    B, T, H, D = 3, 200, 4, 64
    *x, cu_q, _ = inputs([T] * B, [0] * B, H, H, D, torch.bfloat16, seed=11)
    out = forgetting_attention_packed(*x[:4], cu_q)
    dense = forgetting_attention(*(t.reshape(B, T, H, -1).squeeze(-1) for t in x[:4])).reshape(B * T, H, D)
    e = torch.matmul(torch.ones(1, device="cuda"), x[2].float().abs().amax().reshape(1))
    assert ((out - dense).float().abs() <= 2 * 2.0 ** -8 * e).all()


def test_packed_in_a_graph_and_on_streams():
    """A captured step, replayed with other lengths in the same buffers and with eager work between, and two streams at once."""
    from forgetting_transformer import forgetting_attention_packed
    H, Hk, D = 4, 2, 64
    sets = [inputs(new, [0] * 3, H, Hk, D, torch.bfloat16, seed=20 + i, pad=600 - sum(new)) for i, new in enumerate(([100, 300, 50], [1, 0, 599], [200, 200, 200]))]

    def step(x):
        leaves = [t.detach().requires_grad_() for t in x[:4]]
        out = forgetting_attention_packed(*leaves, x[5])
        return [out.detach(), *torch.autograd.grad(out, leaves, x[4])]

    want = [step(x) for x in sets]
    buf = [t.clone() for t in sets[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(buf)
    for i in (0, 1, 2, 1, 0):
        for b, t in zip(buf, sets[i]):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want[i])), i
        step(sets[(i + 1) % 3])
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for _ in range(3):
        for s, x in zip(streams, sets):
            with torch.cuda.stream(s):
                results.append(step(x))
    torch.cuda.synchronize()
    for i, r in enumerate(results):
        assert all(torch.equal(a, b) for a, b in zip(r, want[i % 2]))


def test_packed_ends_out_of_range():
    """Ends that decrease or lie outside the tensors name rows inside them all the same; the sequences in front are right."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, _ = inputs([100, 150, 50], [0] * 3, 2, 2, 32, torch.bfloat16, seed=30)
    want = forgetting_attention_packed(*x[:4], cu_q)
    for bad in ([0, 100, 250, 2 ** 31 - 1], [-7, 100, 250, 300], [0, 100, 250, 249], [0, 100, -5, -6]):
        leaves = [t.detach().requires_grad_() for t in x[:4]]
        out = forgetting_attention_packed(*leaves, torch.tensor(bad, dtype=torch.int32, device="cuda"))
        torch.autograd.grad(out, leaves, x[4])
        assert torch.equal(out[:100], want[:100]), bad
    torch.cuda.synchronize()


def test_packed_nothing_to_do():
    from forgetting_transformer import forgetting_attention_packed
    z = lambda *s: torch.zeros(*s, device="cuda")
    cu = torch.zeros(2, dtype=torch.int32, device="cuda")
    for T, N in ((0, 0), (5, 0), (0, 7)):
        q, k, f = z(T, 4, 64).bfloat16().requires_grad_(), z(N, 2, 64).bfloat16().requires_grad_(), z(N, 4).requires_grad_()
        out = forgetting_attention_packed(q, k, k, f, cu, cu)
        assert out.shape == (T, 4, 64) and not out.any()
        for g, t in zip(torch.autograd.grad(out, (q, k, f), torch.ones_like(out)), (q, k, f)):
            assert g.shape == t.shape and not g.any()
    # all places belong to nobody
    q = torch.full((300, 4, 64), float("nan"), device="cuda").bfloat16().requires_grad_()
    f = z(300, 4).requires_grad_()
    out = forgetting_attention_packed(q, q, q, f, cu)
    assert not out.any() and all(not g.any() for g in torch.autograd.grad(out, (q, f), torch.ones_like(out)))


def test_packed_copies_what_the_kernels_do_not_take():
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, _ = inputs([100, 33], [0, 0], 2, 2, 32, torch.float16, seed=40)
    want = forgetting_attention_packed(*x[:4], cu_q)
    odd = [torch.cat([t[..., :1], t], -1)[..., 1:] for t in x[:3]]              # 2-byte aligned rows
    one = x[1][:1].expand(133, -1, -1)                                          # tokens that lie on each other
    assert torch.equal(forgetting_attention_packed(*odd, x[3].t().contiguous().t(), torch.stack([cu_q, cu_q], 1)[:, 0]), want)
    leaves = [t.detach().requires_grad_() for t in (x[0], one, x[2], x[3])]
    out = forgetting_attention_packed(*leaves, cu_q)
    check((x[0], one, x[2], x[3], x[4]), cu_q, cu_q, 32 ** -0.5, [out.detach(), *torch.autograd.grad(out, leaves, x[4].transpose(1, 2).contiguous().transpose(1, 2))], torch.float16)


def test_packed_refusals():
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([10, 20], [0, 0], 4, 2, 64, torch.bfloat16)
    q, k, v, f = x[:4]
    for bad in (dict(q=q[0]), dict(q=q.float()), dict(q=q.half()), dict(q=q[..., :48], k=k[..., :48], v=v[..., :48]), dict(v=v[:-1]), dict(k=k[:, :1]), dict(f=f.double()), dict(f=f[:, :2]),
                dict(cu=cu_q.long()), dict(cu=cu_q[:1]), dict(cu=cu_q[None]), dict(cu_k=cu_q[:2]), dict(q=q[:20]), dict(q=q[:, :3], f=f[:, :3])):
        a = {**dict(q=q, k=k, v=v, f=f, cu=cu_q, cu_k=None), **bad}
        with pytest.raises(AssertionError):
            forgetting_attention_packed(a["q"], a["k"], a["v"], a["f"], a["cu"], a["cu_k"])
    leaves = [t.detach().requires_grad_() for t in (q, k, v, f)]
    out = forgetting_attention_packed(*leaves, cu_q)
    with pytest.raises(RuntimeError, match="no second derivative"):
        torch.autograd.grad(out, leaves, x[4].requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda q: forgetting_attention_packed(q, k, v, f, cu_q))(q[None])


def test_packed_of_more_than_four_gi_elements():
    """Sequences whose elements lie behind 2**32: the same bits as from a call of their own."""
    from forgetting_transformer import forgetting_attention_packed
    H, D, n, B = 128, 128, 256, 1026
    T, tail = B * n, 2 * n
    g = torch.Generator(device="cuda").manual_seed(41)
    small = [torch.randn(tail, H, D, generator=g, device="cuda").bfloat16() for _ in range(4)]
    gates = -torch.rand(tail, H, generator=g, device="cuda")
    small.insert(3, gates)

    def step(q, k, v, f, do):
        cu = torch.arange(0, len(q) + 1, n, dtype=torch.int32, device="cuda")
        leaves = [t.detach().requires_grad_() for t in (q, k, v, f)]
        out = forgetting_attention_packed(*leaves, cu)
        return [t[-tail:].clone() for t in (out.detach(), *torch.autograd.grad(out, leaves, do))]

    want = step(*small)
    large = []
    for t in small:
        x = torch.zeros(T, *t.shape[1:], dtype=t.dtype, device="cuda")
        x[-tail:] = t
        large.append(x)
    for a, b in zip(step(*large), want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("new,front,H,Hk,D,dtype,at", [   # `at`: the sequence, the key and the head whose gate is NaN
    ([40, 200, 33], [0, 0, 0], 4, 2, 64, torch.bfloat16, (1, 70, 1)), ([300, 90], [0, 50], 3, 1, 16, torch.float16, (0, 299, 2)),
    ([600, 20, 5], [0, 0, 0], 4, 4, 128, torch.bfloat16, (0, 130, 3)), ([5, 100], [900, 0], 8, 2, 128, torch.float16, (0, 3, 0)),
    ([7, 1, 1], [0, 0, 0], 2, 2, 32, torch.bfloat16, (1, 0, 0)), ([1300, 30], [0, 0], 1, 1, 64, torch.bfloat16, (0, 1000, 0)),
    ([1500, 20], [700, 0], 2, 1, 128, torch.bfloat16, (0, 1900, 1))])
def test_packed_gate_that_is_nan(new, front, H, Hk, D, dtype, at):
    """A NaN in one head's gate of a sequence: what the formulas make of it, and nothing else. Rows behind it are NaN, and every key of the sequence is seen from one of them."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs(new, front, H, Hk, D, dtype, seed=50 + D, lead=2, pad=3)
    b, key, h = at
    r0, rows, k0, keys = cu_q[b].item(), new[b], cu_k[b].item(), new[b] + front[b]

    def step():
        leaves = [t.detach().clone().requires_grad_() for t in x[:4]]
        out = forgetting_attention_packed(*leaves, cu_q, cu_k)
        return [out.detach(), *torch.autograd.grad(out, leaves, x[4])]

    want = step()
    x[3][k0 + key, h] = float("nan")
    got = step()
    first = r0 + max(rows - (keys - key), 0)                # of the rows that see the key
    hk = h // (H // Hk)
    is_nan = [torch.zeros_like(y, dtype=torch.bool) for y in want]
    for i in (0, 1):                                        # o, dq
        is_nan[i][first:r0 + rows, h] = True
    for i in (2, 3):                                        # dk, dv of the key head
        is_nan[i][k0:k0 + keys, hk] = True
    is_nan[4][k0:k0 + keys, h] = True
    for name, y, w, n in zip(("o", "dq", "dk", "dv", "dg"), got, want, is_nan):
        assert torch.equal(torch.isnan(y), n), f"{name}: {torch.isnan(y).sum().item()} NaN, {n.sum().item()} by the formulas"
        assert torch.equal(y[~n], w[~n]), name


@pytest.mark.parametrize("ends,H,Hk,D", [
    ([0, 100, 50, 120], 2, 2, 32), ([0, 100, 250, 90, 95, 240, 300], 3, 1, 64), ([30, -5, 300, 20, 10, 280, 299, 7], 4, 2, 16), ([-1, 0, 2 ** 31 - 1, 5, 9], 1, 1, 128),
    ([0] + [(37 * i) % 301 for i in range(200)], 5, 5, 32), ([0] + [min(i, 299) if i % 50 else 40 for i in range(1500)], 2, 1, 16)])
def test_packed_ends_that_decrease(ends, H, Hk, D):
    """Every sequence begins behind all earlier ends, and ends behind the tensors are left out: the same bits as from ends that are in that order."""
    from forgetting_transformer import forgetting_attention_packed
    *x, _, _ = inputs([300], [0], H, Hk, D, torch.bfloat16, seed=60)
    given = torch.tensor(ends, dtype=torch.int32, device="cuda")
    order = torch.where(given > 300, 0, given).clamp(min=0).cummax(0).values.int()

    def step(*cu):
        leaves = [t.detach().requires_grad_() for t in x[:4]]
        out = forgetting_attention_packed(*leaves, *cu)
        return [out.detach(), *torch.autograd.grad(out, leaves, x[4])]

    for a, b in ((step(given), step(order)), (step(given, order), step(order, order)), (step(order, given), step(order, order))):
        assert all(torch.equal(y, z) for y, z in zip(a, b))


def test_packed_ends_behind_the_tensors():
    """A sequence that ends behind the keys, or behind the queries, holds none, and neither do those that follow; the ones in front are whole."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([40, 200, 33, 5], [0, 90, 20, 7], 4, 2, 64, torch.bfloat16, seed=61)
    ends_q, ends_k = cu_q.tolist(), cu_k.tolist()
    for T, N in ((278, 394), (278, 383), (278, 331), (278, 330), (278, 39), (277, 395), (273, 395), (100, 395), (272, 360), (39, 200)):
        leaves = [t.detach().requires_grad_() for t in (x[0][:T], *(t[:N] for t in x[1:4]))]
        out = forgetting_attention_packed(*leaves, cu_q, cu_k)
        got = [out.detach(), *torch.autograd.grad(out, leaves, x[4][:T])]
        m = [e if e <= T else max(y for y in ends_q if y <= T) for e in ends_q]        # without the ends behind them
        n = [e if e <= N else max(y for y in ends_k if y <= N) for e in ends_k]
        order = [torch.tensor(e, dtype=torch.int32, device="cuda") for e in (m, n)]
        check([t[:len(y)] for t, y in zip(x, (*leaves, out))], *order, 64 ** -0.5, got, torch.bfloat16)


@pytest.mark.parametrize("D,dtype", [(16, torch.float16), (64, torch.bfloat16), (128, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("scale", [-0.2, -1e-3, 0.0, 1e-32, 1e-3, 0.3])
def test_packed_scales_of_long_walks(D, dtype, scale):
    """Scales of either sign and next to none where most steps lie off the diagonal, heads and rows in parts among them. A probability's error relative to itself goes with the size of the scores,
    so the norm of dg is held to 2^-16 for scores of size one and to as much more as they are larger."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([900, 1, 260], [0, 300, 700], 4, 2, D, dtype, seed=70 + D)
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = forgetting_attention_packed(*leaves, cu_q, cu_k, sm_scale=scale)
    wrong, size = check(x, cu_q, cu_k, scale, [out.detach(), *torch.autograd.grad(out, leaves, x[4])], dtype)
    assert wrong <= 2.0 ** -16 * max(1.0, abs(scale) * D ** 0.5) * size


@pytest.mark.parametrize("D,dtype", [(64, torch.float16), (128, torch.bfloat16), (128, torch.float16)])
def test_packed_closed_gates_of_long_walks(D, dtype):
    """Closed gates in interior tiles and at the diagonal; the norm of dg is held too."""
    from forgetting_transformer import forgetting_attention_packed
    *x, cu_q, cu_k = inputs([800, 130], [100, 500], 4, 2, D, dtype, seed=80 + D)
    f = x[3]
    f[60], f[300], f[301, 1], f[700] = -math.inf, torch.finfo(torch.float32).min, -math.inf, -math.inf
    f[900], f[1200:1203, 2] = -math.inf, -math.inf                 # the first gate of a sequence, several in a row
    leaves = [t.detach().requires_grad_() for t in x[:4]]
    out = forgetting_attention_packed(*leaves, cu_q, cu_k)
    wrong, size = check(x, cu_q, cu_k, D ** -0.5, [out.detach(), *torch.autograd.grad(out, leaves, x[4])], dtype)
    assert wrong <= 2.0 ** -16 * size
