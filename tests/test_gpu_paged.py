"""Serving from pages: slots and block tables, the append, attention over the pages, and all of them together against the dense cache.

Tolerance of the attention: half a step of the output's type, and 32-bit arithmetic in front of it: a score is off by the rounding of a dot product of at most
128 terms and of the sum of the gates, together below 2^-17 of |q||k| scale + |bias|, for scores that carry weight below 2^-13 here; the weights are off by as much,
so o by twice that of the largest |v|: 2^-12 max|v|."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference_slots(lengths, new, table, stack, S, T, W):
    """The bookkeeping of a step, request by request; changes its lists."""
    slots, positions, requests, keys, granted, full, at = [-1] * T, [0] * T, [-1] * T, [0] * T, [], False, 0
    for b, n in enumerate(new):
        held, want = -(-lengths[b] // S), -(-(lengths[b] + n) // S)
        ok = at + n <= T and want <= W
        if ok and want > held:
            full = full or want - held > len(stack)
            ok = not full
        if ok:
            table[b][held:want] = [stack.pop() for _ in range(want - held)]
        for i in range(min(n, max(0, T - at))):
            p = lengths[b] + i
            positions[at + i] = p
            if ok:
                slots[at + i], requests[at + i], keys[at + i] = table[b][p // S] * S + p % S, b, p + 1
        at += n
        lengths[b] += n if ok else 0
        granted.append(ok)
    return slots, positions, requests, keys, granted


def state(B, W, P, S, seed, longest=None):
    """Requests that hold pages of a shuffled pool; what is left is the stack."""
    g = torch.Generator().manual_seed(seed)
    pages = torch.randperm(P, generator=g).tolist()
    lengths, table = [], []
    for b in range(B):
        n = int(torch.randint(0, min(longest or W * S, W * S) + 1, (1,), generator=g))
        n = min(n, max(0, len(pages) - (B - b)) * S)
        lengths.append(n)
        row = [pages.pop() for _ in range(-(-n // S))]
        table.append(row + [-1] * (W - len(row)))
    return lengths, table, pages, g


def on_gpu(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,W,P,S,T,most,seed", [(1, 1, 1, 8, 8, 8, 0), (1, 4, 8, 16, 1, 1, 1), (5, 6, 40, 16, 64, 20, 2), (64, 40, 900, 32, 64, 1, 3), (200, 9, 1000, 8, 700, 9, 4),
                                                  (1025, 5, 2500, 16, 3000, 4, 5), (4096, 3, 9000, 8, 5000, 2, 6), (7, 300, 1500, 16, 9000, 4000, 7), (3, 8, 12, 64, 0, 5, 8),
                                                  (40, 8, 90, 8, 400, 30, 9), (2500, 4, 3000, 64, 2500, 3, 10)])
def test_page_slots(B, W, P, S, T, most, seed, in_place):
    from forgetting_transformer import page_slots
    lengths, table, stack, g = state(B, W, P, S, seed, longest=W * S // 2)
    new = torch.randint(0, most + 1, (B,), generator=g).tolist()
    dl, dt = on_gpu(lengths), on_gpu(table)
    dp = on_gpu(stack + [-7] * (P - len(stack)))
    dc = on_gpu([len(stack)])
    s = page_slots(dl, on_gpu(new), dt, dp, dc, page_size=S, max_tokens=T, in_place=in_place)
    want = reference_slots(lengths, new, table, stack, S, T, W)
    assert (s.lengths is dl) == in_place or torch.equal(s.lengths, dl)
    for name, got, ref in zip(("slots", "positions", "requests", "keys", "granted"), (s.slots, s.positions, s.requests, s.keys, s.granted), want):
        assert got.tolist() == ref, name
    assert s.lengths.tolist() == lengths and s.free_count.tolist() == [len(stack)] and dt.tolist() == table
    if in_place:
        assert dl.tolist() == lengths and dc.tolist() == [len(stack)]
    used = [x for x in s.slots.tolist() if x >= 0]
    assert len(set(used)) == len(used)


def test_page_slots_state_out_of_range():
    """Counts, lengths and stacks that no program of this library writes stay inside their buffers."""
    from forgetting_transformer import page_slots
    W, S, P = 4, 16, 6
    free = on_gpu([0, 1, 2, 3, 4, 5])
    s = page_slots(on_gpu([-5, 1000, 3]), on_gpu([1, 1, -4]), on_gpu([[-1] * W] * 3), free, on_gpu([99]), page_size=S, max_tokens=4)
    assert s.slots.tolist() == [5 * S, -1, -1, -1] and s.granted.tolist() == [True, False, True] and s.lengths.tolist() == [1, W * S, 3] and s.free_count.tolist() == [5]
    s = page_slots(on_gpu([0, 0]), on_gpu([2 ** 31 - 1, 2 ** 31 - 1]), on_gpu([[-1] * W] * 2), free, on_gpu([-3]), page_size=S, max_tokens=3)
    assert s.slots.tolist() == [-1] * 3 and s.positions.tolist() == [0, 1, 2] and s.granted.tolist() == [False, False] and s.free_count.tolist() == [0]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("B,W,P,S,seed", [(1, 3, 5, 16, 0), (9, 70, 500, 8, 1), (300, 5, 1200, 16, 2), (4096, 2, 8000, 8, 3)])
def test_page_release(B, W, P, S, seed, in_place):
    from forgetting_transformer import page_release
    lengths, table, stack, g = state(B, W, P, S, seed)
    done = (torch.rand(B, generator=g) < 0.4).tolist()
    dl, dp, dc, dt = on_gpu(lengths), on_gpu(stack + [-7] * (P - len(stack))), on_gpu([len(stack)]), on_gpu(table)
    out_l, out_c = page_release(dl, on_gpu(done, torch.bool), dt, dp, dc, page_size=S, in_place=in_place)
    for b, d in enumerate(done):
        if d:
            stack += table[b][:-(-lengths[b] // S)]
            lengths[b] = 0
    assert out_l.tolist() == lengths and out_c.tolist() == [len(stack)] and dp.tolist()[:len(stack)] == stack and dt.tolist() == table
    assert dp.tolist()[len(stack):] == [-7] * (P - len(stack)) and (out_l is dl or not in_place)


def test_page_release_of_a_full_stack():
    from forgetting_transformer import page_release
    free = on_gpu([3, 2, 1, 0])
    _, count = page_release(on_gpu([64, 64]), on_gpu([True, True], torch.bool), on_gpu([[0, 1, 2, 3]] * 2), free, on_gpu([3]), page_size=16)
    assert free.tolist() == [3, 2, 1, 0] and count.tolist() == [4]


def pool(P, H, S, D, dtype, seed, heads_inside=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (P, S, H, D) if heads_inside else (P, H, S, D)
    k, v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
    f = torch.nn.functional.logsigmoid(torch.randn(shape[:3], generator=g, device="cuda") + 2.0)
    return (k.transpose(1, 2), v.transpose(1, 2), f.transpose(1, 2), g) if heads_inside else (k, v, f, g)


@pytest.mark.parametrize("T,H,D,S,P,dtype,inside", [(1, 1, 16, 8, 2, torch.bfloat16, False), (37, 3, 32, 16, 5, torch.float16, True), (1000, 12, 64, 64, 20, torch.bfloat16, False),
                                                     (513, 5, 128, 32, 17, torch.float16, True)])
def test_paged_append(T, H, D, S, P, dtype, inside):
    from forgetting_transformer import paged_append
    kp, vp, fp, g = pool(P, H, S, D, dtype, 1, inside)
    k, v = (torch.randn(T, H, D, generator=g, device="cuda").to(dtype) for _ in range(2))
    f = -torch.rand(H, T, generator=g, device="cuda").t()          # strided gates
    slots = torch.randperm(P * S, generator=g, device="cuda")[:T]
    slots[::7] = -1
    slots[3::11] = P * S + 5
    want = [t.clone() for t in (kp, vp, fp)]
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < P * S:
            for w, x in zip(want, (k, v, f)):
                w[s // S, :, s % S] = x[t]
    paged_append(k, v, f, kp, vp, fp, slots)
    assert all(torch.equal(a, b) for a, b in zip((kp, vp, fp), want))
    before = kp._version
    wide = torch.randn(T, H, 2 * D + 1, generator=g, device="cuda").to(dtype)[..., 1:D + 1]     # 2-byte aligned rows: copied first
    paged_append(wide, wide, f, kp, vp, fp, slots)
    assert kp._version > before
    t = 1 if T > 1 else None
    if t is not None:
        s = int(slots[t])
        assert torch.equal(kp[s // S, :, s % S], wide[t]) and torch.equal(vp[s // S, :, s % S], wide[t])
    paged_append(k[:0], v[:0], f[:0], kp, vp, fp, slots[:0])


def test_keys_and_values_in_one_pool():
    """Pages of keys and values between each other, (P, 2, H, S, D), as two views."""
    from forgetting_transformer import paged_append, paged_forgetting_attention
    P, H, S, D, T = 6, 3, 16, 64, 70
    kv = torch.zeros(P, 2, H, S, D, dtype=torch.bfloat16, device="cuda")
    f = torch.zeros(P, H, S, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    k, v = (torch.randn(T, H, D, generator=gen, device="cuda").bfloat16() for _ in range(2))
    g = -torch.rand(T, H, generator=gen, device="cuda")
    paged_append(k, v, g, kv[:, 0], kv[:, 1], f, torch.arange(T, device="cuda"))
    apart = [torch.zeros(P, H, S, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)] + [torch.zeros_like(f)]
    paged_append(k, v, g, *apart, torch.arange(T, device="cuda"))
    assert torch.equal(kv[:, 0], apart[0]) and torch.equal(kv[:, 1], apart[1]) and torch.equal(f, apart[2])
    table, n = on_gpu([list(range(P))]), on_gpu([T])
    assert torch.equal(paged_forgetting_attention(k[:1], kv[:, 0], kv[:, 1], f, table, n), paged_forgetting_attention(k[:1], *apart, table, n))


def attention_reference(q, kp, vp, fp, table, lengths, requests, scale):
    P, H, S, D = kp.shape
    out = torch.zeros_like(q, dtype=torch.float64)
    for b, n in enumerate(lengths):
        r = b if requests is None else requests[b]
        n = min(n, len(table[0]) * S)
        if not 0 <= r < len(table) or n <= 0:
            continue
        at = torch.arange(n, device="cuda")
        pages = torch.tensor(table[r], device="cuda")[at // S]
        here = (pages >= 0) & (pages < P)
        if not here.any():
            continue
        page, row = pages.clamp(0, P - 1), at % S
        k, v, f = (t[page, :, row].double().transpose(0, 1) for t in (kp, vp, fp))     # (H, n, D), (H, n)
        f = torch.where(here, f, 0.0)
        # of the gates behind each key (not the sum with its own less its own, which a very negative gate would swallow)
        behind = torch.cat([f[:, 1:], f.new_zeros(H, 1)], -1).flip(-1).cumsum(-1).flip(-1)
        s = (k * q[b].double()[:, None]).sum(-1) * scale + behind
        s = torch.where(here, s, float("-inf"))
        p = torch.softmax(s, -1)
        out[b] = torch.where((p > 0)[..., None], p[..., None] * v, 0.0).sum(1)
    return out


def check_attention(got, want, vp, dtype):
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -12 * vp[torch.isfinite(vp)].double().abs().max()
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"{(err / bound).max().item():.3f} of its bound"


CASES = [  # B, H, D, S, W, lengths, dtype, heads inside
    (1, 1, 16, 8, 1, [1], torch.bfloat16, False), (3, 2, 32, 8, 4, [0, 1, 32], torch.float16, False), (4, 3, 64, 16, 20, [5, 16, 17, 320], torch.bfloat16, True),
    (2, 12, 64, 16, 100, [1500, 1], torch.bfloat16, False), (2, 4, 128, 64, 40, [2560, 2499], torch.float16, True), (5, 2, 16, 16, 200, [3200, 0, 7, 1024, 1025], torch.float16, False),
    (1, 2, 128, 4096, 3, [9001], torch.bfloat16, False), (70, 2, 32, 32, 30, None, torch.bfloat16, False), (130, 1, 64, 8, 90, None, torch.float16, True),
    (1, 1, 128, 32, 700, [22400], torch.bfloat16, False), (6, 16, 128, 256, 4, None, torch.bfloat16, False), (300, 3, 16, 8, 40, None, torch.bfloat16, False),
    (2, 2, 32, 8, 3000, [24000, 200], torch.bfloat16, False), (1100, 2, 64, 16, 40, None, torch.bfloat16, False), (256, 1, 128, 16, 100, None, torch.float16, True)]


@pytest.mark.parametrize("B,H,D,S,W,lengths,dtype,inside", CASES)
def test_paged_attention(B, H, D, S, W, lengths, dtype, inside):
    from forgetting_transformer import paged_forgetting_attention
    g = torch.Generator().manual_seed(B + W)
    if lengths is None:
        lengths = (torch.rand(B, generator=g) ** 3 * (W * S + 1)).long().tolist()
        lengths[0], lengths[-1] = 0, W * S
    P = sum(-(-n // S) for n in lengths) + 2
    kp, vp, fp, gen = pool(P, H, S, D, dtype, 2, inside)
    kp[P - 1], vp[P - 1], fp[P - 1] = float("nan"), float("nan"), float("nan")     # a page that nobody holds
    ids = torch.randperm(P - 1, generator=g).tolist()
    table = [[ids.pop() for _ in range(-(-n // S))] for n in lengths]
    for row, n in zip(table, lengths):                                             # what lies behind the last token of a page may be anything
        if n % S:
            kp[row[-1], :, n % S:], vp[row[-1], :, n % S:], fp[row[-1], :, n % S:] = float("nan"), float("inf"), float("nan")
    table = [row + [P - 1] * (W - len(row)) for row in table]
    q = torch.randn(B, H, D, generator=gen, device="cuda").to(dtype)
    args = (q, kp, vp, fp, on_gpu(table), on_gpu(lengths))
    out = paged_forgetting_attention(*args)
    assert out.dtype == dtype and out.shape == q.shape
    want = attention_reference(q, kp, vp, fp, table, lengths, None, D ** -0.5)
    check_attention(out, want, vp, dtype)
    assert torch.equal(paged_forgetting_attention(*args), out)
    if max(lengths) < W * S:                                                        # fewer launches and scratch, other pieces perhaps
        check_attention(paged_forgetting_attention(*args, max_length=max(max(lengths), 1)), want, vp, dtype)
    order = torch.randint(-1, B, (B + 3,), generator=g).tolist()                    # some requests twice, some rows without one
    seen = [lengths[r] // 2 + 1 if r >= 0 else 5 for r in order]
    seen = [min(n, lengths[r]) if r >= 0 else n for n, r in zip(seen, order)]
    q2 = torch.randn(B + 3, H, D, generator=gen, device="cuda").to(dtype)
    out = paged_forgetting_attention(q2, kp, vp, fp, args[4], on_gpu(seen), requests=on_gpu(order), sm_scale=0.3)
    check_attention(out, attention_reference(q2, kp, vp, fp, table, seen, order, 0.3), vp, dtype)


def test_paged_attention_gates_that_close():
    """Gates of minus infinity cut everything in front of them off, whatever pieces and runs they fall into; very negative ones as well."""
    from forgetting_transformer import paged_forgetting_attention
    H, D, S, W = 2, 64, 16, 300
    for seed, (n, cuts, value) in enumerate([(4800, [4799], float("-inf")), (4800, [100, 2500, 4300], float("-inf")), (1000, [0, 999], float("-inf")), (4000, [3100], -3.0e38),
                                             (4800, list(range(4000)), -1.0e4)]):
        kp, vp, fp, gen = pool(W + 1, H, S, D, torch.bfloat16, seed)
        table = torch.randperm(W, generator=torch.Generator().manual_seed(seed)).tolist()
        for c in cuts:
            fp[table[c // S], :, c % S] = value
        q = torch.randn(1, H, D, generator=gen, device="cuda").bfloat16()
        out = paged_forgetting_attention(q, kp, vp, fp, on_gpu([table]), on_gpu([n]))
        check_attention(out, attention_reference(q, kp, vp, fp, [table], [n], None, D ** -0.5), vp, torch.bfloat16)
        if value == float("-inf"):
            vp[[p for p in range(W + 1) if p not in table[max(cuts) // S:]]] = 0.0          # keys in front of the last closed gate have no weight
            assert torch.equal(paged_forgetting_attention(q, kp, vp, fp, on_gpu([table]), on_gpu([n])), out)


def test_paged_attention_pages_outside_the_pool():
    """Table entries that name no page: their keys are left out; a row of nothing else gives zeros."""
    from forgetting_transformer import paged_forgetting_attention
    H, D, S, W, P = 3, 32, 8, 70, 64
    kp, vp, fp, gen = pool(P, H, S, D, torch.bfloat16, 3)
    vp[0] = float("nan")                                                            # page 0 is what a missing page's address falls back to
    g = torch.Generator().manual_seed(1)
    table = [[1 + int(x) for x in torch.randperm(P - 1, generator=g)] + [1] * (W - P + 1) for _ in range(3)]
    for r, bad in ((0, [0, 5, 30]), (1, list(range(W))), (2, [W - 1])):
        for i in bad:
            table[r][i] = [-1, P, 2 ** 31 - 1, -2 ** 31][i % 4]
    q = torch.randn(3, H, D, generator=gen, device="cuda").bfloat16()
    lengths = [W * S, W * S - 3, W * S]
    out = paged_forgetting_attention(q, kp, vp, fp, on_gpu(table), on_gpu(lengths))
    check_attention(out, attention_reference(q, kp, vp, fp, table, lengths, None, D ** -0.5), vp, torch.bfloat16)
    assert out[1].abs().max() == 0
    out = paged_forgetting_attention(q, kp, vp, fp, on_gpu(table), on_gpu([2 ** 31 - 1, -7, 0]))       # lengths beyond the table are cut to it
    assert torch.equal(out[0], paged_forgetting_attention(q, kp, vp, fp, on_gpu(table), on_gpu(lengths))[0]) and out[1:].abs().max() == 0


def test_paged_attention_views_beyond_32_bits():
    """A pool whose pages lie further apart than 2^31 elements in all, and requests that use the last of them."""
    from forgetting_transformer import paged_append, paged_forgetting_attention
    P, H, S, D = 520, 2, 16, 64
    gap = 1 << 22                                                                    # elements between pages: the last one starts beyond 2^31
    k_mem, v_mem = (torch.empty(P * gap, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    kp, vp = (m.as_strided((P, H, S, D), (gap, S * D, D, 1)) for m in (k_mem, v_mem))
    fp = torch.zeros(P, H, S, device="cuda")
    gen = torch.Generator(device="cuda").manual_seed(0)
    n = 100
    k, v = (torch.randn(n, H, D, generator=gen, device="cuda").bfloat16() for _ in range(2))
    f = -torch.rand(n, H, generator=gen, device="cuda")
    table = [P - 1 - i for i in range(7)]
    at = torch.arange(n, device="cuda")
    paged_append(k, v, f, kp, vp, fp, torch.tensor(table, device="cuda")[at // S] * S + at % S)
    q = torch.randn(1, H, D, generator=gen, device="cuda").bfloat16()
    out = paged_forgetting_attention(q, kp, vp, fp, on_gpu([table]), on_gpu([n]))
    s = (k.double() * q.double()).sum(-1) * D ** -0.5 + f.double().flip(0).cumsum(0).flip(0) - f.double()
    want = (torch.softmax(s, 0)[..., None] * v.double()).sum(0)[None]
    check_attention(out, want, v, torch.bfloat16)


def test_refusals_on_the_gpu():
    from forgetting_transformer import page_slots, paged_append, paged_forgetting_attention
    kp, vp, fp, _ = pool(4, 2, 16, 64, torch.bfloat16, 0)
    table, lengths = on_gpu([[0, 1], [2, 3]]), on_gpu([20, 5])
    q = torch.zeros(2, 2, 64, device="cuda").bfloat16()
    t = lambda *s: torch.zeros(*s, device="cuda")
    for bad in (dict(q=q.half()), dict(q=q[:, :1]), dict(q=q[:1]), dict(table=table.long()), dict(table=table[0]), dict(lengths=lengths.long()), dict(lengths=lengths[:1]),
                dict(requests=lengths[:1]), dict(max_length=0), dict(fp=fp[:3])):
        a = {**dict(q=q, fp=fp, table=table, lengths=lengths, requests=None, max_length=None), **bad}
        with pytest.raises(AssertionError):
            paged_forgetting_attention(a["q"], kp, vp, a["fp"], a["table"], a["lengths"], requests=a["requests"], max_length=a["max_length"])
    with pytest.raises(RuntimeError, match="does not take"):
        paged_forgetting_attention(q.clone().requires_grad_(), kp, vp, fp, table, lengths)
    k, f, slots = t(3, 2, 64).bfloat16(), t(3, 2), torch.arange(3, device="cuda")
    for bad in (dict(k=k[:2]), dict(f=f.t()), dict(f=f.half()), dict(slots=slots.int()), dict(slots=slots[:2])):
        a = {**dict(k=k, f=f, slots=slots), **bad}
        with pytest.raises(AssertionError):
            paged_append(a["k"], k, a["f"], kp, vp, fp, a["slots"])
    for bad in ((kp[0].transpose(0, 1)[:3], k, kp), (k, k, kp[:1].expand(4, 2, 16, 64)), (k.clone().requires_grad_(), k, kp), (k, k, vp)):   # reads what it writes; pages that lie on each other; a graph; keys and values in one place
        with pytest.raises(RuntimeError, match="does not take"):
            paged_append(bad[0], bad[1], f, bad[2], vp, fp, slots)
    free, count = on_gpu([0, 1, 2, 3]), on_gpu([4])
    with pytest.raises(RuntimeError, match="does not take"):
        page_slots(lengths, lengths, table, free, free[:1], page_size=16, max_tokens=4)                    # the stack and its count in one place
    with pytest.raises(RuntimeError, match="does not take"):
        page_slots(lengths, lengths, table, free, count, page_size=16, max_tokens=4, in_place=True)        # reads the new tokens where it writes the lengths
    mixed = on_gpu([[7, 0, 1], [8, 2, 3]])
    with pytest.raises(RuntimeError, match="does not take"):
        page_slots(lengths, mixed.view(-1)[:2], mixed[:, :2], free, count, page_size=16, max_tokens=4)     # reads the new tokens where it writes the table
    with pytest.raises(AssertionError):
        page_slots(lengths, lengths, table[:, :1].expand(2, 2), free, count, page_size=16, max_tokens=4)


def test_serving_steps_equal_the_dense_operator():
    """Requests that come, generate and go, through rotation, pages and attention, against the dense operator on each request's own tokens."""
    import forgetting_transformer as ft
    H, D, S, R = 3, 64, 16, 4
    gen = torch.Generator(device="cuda").manual_seed(0)
    host = torch.Generator().manual_seed(0)
    cache = ft.PagedFgateCache(2, H, D, num_pages=40, max_requests=R, max_length=200, page_size=S)
    assert len(cache) == 2
    freq = ft.rotary_frequencies(D, device="cuda")
    wq, wk = (torch.rand(H * D, generator=gen, device="cuda") + 0.5 for _ in range(2))
    stream = [[[], [], []] for _ in range(R)]                       # what each request has fed, layer 1: keys, values, gates
    for step in range(14):
        if step in (6, 10):                                          # two requests end, others take their places
            done = torch.zeros(R, dtype=torch.bool, device="cuda")
            done[step % R] = True
            cache.release(done)
            stream[step % R] = [[], [], []]
        new = torch.randint(0, 3, (R,), generator=host)
        if step in (0, 7):
            new = torch.randint(10, 60, (R,), generator=host)
        T = int(new.sum())
        s = cache.schedule(new.to(torch.int32).cuda(), T + 2)        # two places stay empty
        assert s.granted.all() and s.lengths is cache.lengths
        rnd = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
        q0, k0, v = (rnd(1, T + 2, H, D).bfloat16() for _ in range(3))
        f = torch.nn.functional.logsigmoid(rnd(T + 2, H) + 1.0)
        q, k = ft.qk_norm_rotary(q0, k0, wq, wk, freq, positions=s.positions[None])
        cache.update(k[0], v[0], f, 1)
        out = cache.attend(q[0], 1)
        assert out[T:].abs().max() == 0
        at = 0
        for b, n in enumerate(new.tolist()):
            if n == 0:
                continue
            for store, t in zip(stream[b], (k[0], v[0], f)):
                store.append(t[at:at + n].clone())
            kk, vv, ff = (torch.cat(x)[None] for x in stream[b])
            want = ft.forgetting_attention(q[:, at:at + n], kk, vv, ff)[0]
            # both are within half a step and the operator's bar of the exact result; against 64 bits:
            s64 = torch.einsum("nhd,mhd->hnm", q[0, at:at + n].double(), kk[0].double()) / D ** 0.5
            c = ff[0].double().cumsum(0).t()
            N = kk.shape[1]
            s64 = s64 + c[:, N - n:, None] - c[:, None, :]
            s64 = s64.masked_fill(torch.ones(n, N, device="cuda").tril(N - n) == 0, float("-inf"))
            exact = torch.einsum("hnm,mhd->nhd", torch.softmax(s64, -1), vv[0].double())
            check_attention(out[at:at + n], exact, vv, torch.bfloat16)
            assert (want.double() - out[at:at + n].double()).abs().max() <= 2e-2 * exact.abs().max()
            at += n
    assert int(cache.free_count) == 40 - sum(-(-int(n) // S) for n in cache.lengths.tolist())


def test_a_captured_step_replays():
    """schedule, update and attend of one token per request captured once and replayed: every replay as the eager step."""
    import forgetting_transformer as ft
    H, D, R = 2, 64, 5

    def fresh():
        c = ft.PagedFgateCache(1, H, D, num_pages=60, max_requests=R, max_length=160, page_size=8)
        g = torch.Generator(device="cuda").manual_seed(3)
        n = torch.tensor([3, 40, 0, 100, 7], dtype=torch.int32, device="cuda")
        c.schedule(n, 150)
        x = [torch.randn(150, H, D, generator=g, device="cuda").bfloat16() for _ in range(2)]
        c.update(*x, -torch.rand(150, H, generator=g, device="cuda"), 0)
        return c

    def step(c, new, q, k, v, f):
        c.schedule(new, R)
        c.update(k, v, f, 0)
        return c.attend(q, 0)

    g = torch.Generator(device="cuda").manual_seed(4)
    sets = []
    for i in range(20):
        new = torch.ones(R, dtype=torch.int32, device="cuda")
        new[i % R] = 0
        sets.append([new, *(torch.randn(R, H, D, generator=g, device="cuda").bfloat16() for _ in range(3)), -torch.rand(R, H, generator=g, device="cuda")])
    a = fresh()
    eager = [step(a, *s).clone() for s in sets]
    b = fresh()
    static = [t.clone() for t in sets[0]]
    static[0].zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(b, *static)                                             # a warm-up step that brings no token
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(b, *static)
    for s, want in zip(sets, eager):
        for dst, src in zip(static, s):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        torch.randn(1 << 20, device="cuda").sum().item()
        assert torch.equal(out, want)
    assert torch.equal(a.lengths, b.lengths) and torch.equal(a.block_table, b.block_table) and torch.equal(a.free_count, b.free_count)


def test_lengths_cut_by_max_length():
    from forgetting_transformer import paged_forgetting_attention
    kp, vp, fp, gen = pool(40, 2, 16, 64, torch.float16, 5)
    table = on_gpu([list(range(20)), list(range(20, 40))])
    q = torch.randn(2, 2, 64, generator=gen, device="cuda").half()
    for most in (1, 17, 200, 320, 4000):
        a = paged_forgetting_attention(q, kp, vp, fp, table, on_gpu([320, 100]), max_length=most)
        want = attention_reference(q, kp, vp, fp, table.tolist(), [min(320, most), min(100, most)], None, 64 ** -0.5)
        check_attention(a, want, vp, torch.float16)


def test_steps_in_inference_mode():
    """A cache made and used in inference mode, and one made outside that a step in inference mode writes to."""
    import forgetting_transformer as ft
    freq = ft.rotary_frequencies(32, device="cuda")

    def make():
        return ft.PagedFgateCache(1, 2, 32, num_pages=8, max_requests=3, max_length=40, page_size=8)

    def steps(c):
        g = torch.Generator(device="cuda").manual_seed(0)
        out = []
        for n in ([5, 0, 9], [1, 1, 1], [0, 2, 1]):
            s = c.schedule(on_gpu(n), sum(n))
            q, k, v = (torch.randn(1, sum(n), 2, 32, generator=g, device="cuda").bfloat16() for _ in range(3))
            q, k = ft.qk_norm_rotary(q, k, torch.ones(32, device="cuda"), torch.ones(32, device="cuda"), freq, positions=s.positions[None])
            c.update(k[0], v[0], -torch.rand(sum(n), 2, generator=g, device="cuda"), 0)
            out.append(c.attend(q[0], 0))
        c.release(torch.tensor([True, False, True], device="cuda"))
        return out + [c.lengths.clone(), c.free_count.clone()]

    want = steps(make())
    outside = make()
    with torch.inference_mode():
        inside = steps(make())
        mixed = steps(outside)
    for got in (inside, mixed):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_c_entries():
    """The C entry points on raw pointers: rows that are fewer than the table's requests, and the state of the pages written in place."""
    import ctypes as C
    from forgetting_transformer import paged_forgetting_attention
    from forgetting_transformer.ops import _lib
    lib = _lib.load()
    kp, vp, fp, gen = pool(12, 2, 16, 64, torch.bfloat16, 6)
    view = lambda t: _lib.View(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))
    pages = _lib.Pages(12, 2, 16, 64, 0, view(kp), view(vp), fp.data_ptr(), *fp.stride())
    table, lengths = on_gpu([[0, 1, 2, 3], [4, 5, 6, 7], [8, 9, 10, 11]]), on_gpu([50, 3, 0])
    q = torch.randn(2, 2, 64, generator=gen, device="cuda").bfloat16()
    out = torch.full_like(q, 7.0)
    flat = lambda t: _lib.View(t.data_ptr(), t.stride(0), t.stride(1), 8)
    n = C.c_int64()
    assert lib.fox_paged_decode_workspace_bytes(2, 2, 64, 64, C.byref(n)) == 0
    ws = torch.empty(max(n.value, 16), dtype=torch.uint8, device="cuda")
    args = _lib.PagedDecodeArgs(pages, 2, 3, 4, 0, flat(q), flat(out), table.data_ptr(), 4, lengths.data_ptr(), None, 0.125, ws.data_ptr(), n.value)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    _lib.check(lib.fox_paged_decode(C.byref(args), stream), "fox_paged_decode")
    assert torch.equal(out, paged_forgetting_attention(q, kp, vp, fp, table[:2], lengths[:2]))

    free, count, new = on_gpu([9, 8, 7, 6, 5]), on_gpu([5]), on_gpu([20, 0, 4000])
    state = on_gpu([10, 5, 0])
    T = 1500                                                              # more than a workgroup's tokens: the state has a launch of its own
    slots, pos = (torch.empty(T, dtype=torch.int64, device="cuda") for _ in range(2))
    req, keys = (torch.empty(T, dtype=torch.int32, device="cuda") for _ in range(2))
    granted = torch.empty(3, dtype=torch.bool, device="cuda")
    small = table.clone()
    a = _lib.PageSlotsArgs(3, 4, 5, 16, T, state.data_ptr(), new.data_ptr(), small.data_ptr(), 4, free.data_ptr(), count.data_ptr(), slots.data_ptr(), pos.data_ptr(),
                           req.data_ptr(), keys.data_ptr(), state.data_ptr(), count.data_ptr(), granted.data_ptr())
    _lib.check(lib.fox_page_slots(C.byref(a), stream), "fox_page_slots")
    assert state.tolist() == [30, 5, 0] and count.tolist() == [4] and granted.tolist() == [True, True, False]
    assert slots.tolist()[:20] == [10 + i if i < 6 else 5 * 16 + i - 6 for i in range(20)] and set(slots.tolist()[20:]) == {-1}
    assert small.tolist()[0] == [0, 5, 2, 3] and keys.tolist()[:20] == list(range(11, 31)) and req.tolist()[20:] == [-1] * 1480


def test_limits_are_assertions():
    """Page sizes and widths that no kernel takes are refused like any wrong argument, on the GPU as on the CPU, before anything is written."""
    from forgetting_transformer import page_release, page_slots, paged_append, paged_forgetting_attention
    lengths, free, count = on_gpu([0, 0]), on_gpu([0, 1, 2, 3]), on_gpu([4])
    done = torch.tensor([True, False], device="cuda")
    wide = torch.zeros(1, 1 << 27, dtype=torch.int32, device="cuda")
    for table, size in ((on_gpu([[0, 1], [2, 3]]), 4), (on_gpu([[0, 1], [2, 3]]), 24), (on_gpu([[0, 1], [2, 3]]), 8192), (wide, 16)):
        state = (lengths[:len(table)], lengths[:len(table)] + 1, table, free, count)
        with pytest.raises(AssertionError):
            page_slots(*state, page_size=size, max_tokens=4)
        with pytest.raises(AssertionError):
            page_release(state[0], done[:len(table)], *state[2:], page_size=size)
    for size in (4, 24, 8192):
        kp, vp, fp, _ = pool(3, 1, size, 16, torch.bfloat16, 0)
        x = torch.zeros(2, 1, 16, device="cuda").bfloat16()
        with pytest.raises(AssertionError):
            paged_append(x, x, torch.zeros(2, 1, device="cuda"), kp, vp, fp, torch.arange(2, device="cuda"))
        with pytest.raises(AssertionError):
            paged_forgetting_attention(x, kp, vp, fp, on_gpu([[0], [1]]), on_gpu([1, 1]))


@pytest.mark.parametrize("which", ["pages", "heads", "tokens"])
def test_append_refuses_pages_that_lie_on_each_other(which):
    """Keys and values that share memory without beginning at one place."""
    from forgetting_transformer import paged_append
    H, D, S, P, T = 2, 64, 16, 6, 40
    k, f, slots = torch.ones(T, H, D, device="cuda").bfloat16(), torch.zeros(T, H, device="cuda"), torch.arange(T, device="cuda")
    zeros = lambda *s: torch.zeros(s, dtype=torch.bfloat16, device="cuda")
    x = {"pages": lambda: zeros(P + 1, H, S, D), "heads": lambda: zeros(P, H + 1, S, D), "tokens": lambda: zeros(P, S + 2, H, D).transpose(1, 2)}[which]()
    kp, vp = {"pages": lambda: (x[:-1], x[1:]), "heads": lambda: (x[:, 1:], x[:, :-1]), "tokens": lambda: (x[:, :, :S], x[:, :, 2:])}[which]()
    with pytest.raises(RuntimeError, match="may not overlap"):
        paged_append(k, k, f, kp, vp, torch.zeros(P, H, S, device="cuda"), slots)
    assert not x.any()
