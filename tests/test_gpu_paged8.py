"""Pages of 8-bit keys and values: the quantising append and the gather, both exact, attention over the pages, and all of them together.

Append and gather are compared for equality: their roundings are fixed.  Tolerance of the attention: half a step of the output's type, and 32-bit arithmetic in front of it.  Codes are
exact in bf16 and the products are summed in 32 bits; a score is off by the rounding of a dot product of at most 128 terms, its scale and the sum of the gates, together below 2^-13 for scores that
carry weight here (as with 16-bit pages), a weight by as much and by the 2^-16 that two bf16 parts leave, so o by 2^-12 of the largest |v|."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

CODES = {"e4m3": (torch.float8_e4m3fn, 448.0), "int8": (torch.int8, 127.0)}


def nearest(x, codes):
    """64-bit values to the nearest code's value, ties to the even one; infinities to the largest, NaN to itself or 0."""
    largest = CODES[codes][1]
    if codes == "int8":
        return torch.nan_to_num(x, nan=0.0, posinf=largest, neginf=-largest).clamp(-largest, largest).round()
    x = x.clamp(-largest, largest)
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))) / 8
    return (x / step).round() * step


def pool(P, H, Hk, S, D, codes, seed, layout="apart", power=True):
    """Pages with every code but NaN, scales (powers of two or not) and gates."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    G = min(S, 16)
    shape = {"apart": (2, P, Hk, S, D), "between": (P, 2, Hk, S, D), "inside": (2, P, S, Hk, D)}[layout]
    raw = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)
    if codes == "e4m3":
        raw = torch.where(raw & 127 == 127, raw & 128, raw)
    else:
        raw = torch.where(raw == 128, 127, raw)
    raw = raw.view(CODES[codes][0])
    k, v = {"apart": lambda: (raw[0], raw[1]), "between": lambda: (raw[:, 0], raw[:, 1]), "inside": lambda: (raw[0].transpose(1, 2), raw[1].transpose(1, 2))}[layout]()
    sc = torch.rand(P, S // G, 2, Hk, generator=g, device="cuda") * 4 - 9
    sc = torch.exp2(sc.round() if power else sc)
    ks, vs = (sc[:, :, i].transpose(1, 2) for i in range(2))            # strided, keys' and values' between each other
    f = torch.nn.functional.logsigmoid(torch.randn(P, H, S, generator=g, device="cuda") + 2.0)
    return k, v, ks, vs, f, g


def as_values(pages):
    return pages.double()


def reference_append(k, v, f, pages, slots, codes):
    """Token runs one by one; changes 64-bit copies of (k codes, v codes, k scales, v scales, gates)."""
    kp, vp, ks, vs, fp = (as_values(t).clone() for t in pages)
    P, Hk, S, D = kp.shape
    G = min(S, 16)
    t = 0
    while t < len(slots):
        s = slots[t]
        if not 0 <= s < P * S:
            t += 1
            continue
        n = 1
        while t + n < len(slots) and slots[t + n] == s + n and (s + n) % G:
            n += 1
        page, at = s // S, s % S
        block, row = at // G, at % G
        for x, codes_at, scales in ((k, kp, ks), (v, vp, vs)):
            y = x[t:t + n].double().transpose(0, 1)                     # (Hk, n, D)
            amax = torch.where(torch.isfinite(y), y.abs(), 0.0).amax((1, 2))
            need = torch.exp2(torch.ceil(torch.log2((amax / CODES[codes][1]).clamp(min=2.0 ** -126)))).clamp(min=2.0 ** -126)
            old = scales[page, :, block]
            new = torch.maximum(need, old) if row else need
            if row:
                ratio = (old.float() / new.float()).double()             # the ratio and the product are rounded to 32 bits
                held = codes_at[page, :, at - row:at]
                again = nearest((held * ratio[:, None, None]).float().double(), codes)
                codes_at[page, :, at - row:at] = torch.where((new != old)[:, None, None], again, held)
            inv = (1.0 / new.float())
            codes_at[page, :, at:at + n] = nearest((y.float() * inv[:, None, None]).double(), codes)
            scales[page, :, block] = new
        fp[page, :, at:at + n] = f[t:t + n].double().t()
        t += n
    return kp, vp, ks, vs, fp


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=12345.0), torch.nan_to_num(b, nan=12345.0))


def run_slots(runs):   # of (first slot, tokens); a negative one: tokens without a slot
    return [s + i if s >= 0 else -1 for s, n in runs for i in range(n)]


APPENDS = [  # H, Hk, D, S, P, codes, dtype, layout, runs of slots
    (1, 1, 16, 8, 2, "e4m3", torch.bfloat16, "apart", [(3, 1)]),
    (2, 2, 32, 8, 5, "int8", torch.float16, "between", [(0, 8), (9, 7), (31, 1), (16, 3)]),
    (12, 12, 64, 16, 40, "int8", torch.float16, "apart", [(16 * i + (7 * i) % 16, 1) for i in range(39)]),
    (12, 4, 64, 16, 70, "e4m3", torch.bfloat16, "inside", [(0, 200), (-1, 5), (16 * 13 + 5, 500), (16 * 50, 1), (99999, 1), (16 * 60 + 15, 17)]),
    (16, 4, 128, 64, 30, "e4m3", torch.bfloat16, "apart", [(64 * 3, 700), (7, 33), (64 * 20 + 63, 400)]),
    (5, 1, 128, 32, 40, "int8", torch.bfloat16, "between", [(32 * 2 + 1, 333), (32 * 20, 128)]),
    (3, 3, 16, 4096, 2, "int8", torch.float16, "inside", [(1000, 3000), (5, 20), (4097, 1)]),
    (32, 8, 128, 16, 300, "e4m3", torch.float16, "apart", [(16 * i + (5 * i) % 16, 1) for i in range(290)]),
    (8, 8, 32, 128, 64, "e4m3", torch.bfloat16, "apart", [(0, 128 * 63)]),
]


@pytest.mark.parametrize("H,Hk,D,S,P,codes,dtype,layout,runs", APPENDS)
@pytest.mark.parametrize("power", [True, False])
def test_append(H, Hk, D, S, P, codes, dtype, layout, runs, power):
    from forgetting_transformer import paged_append_8bit
    *pages, g = pool(P, H, Hk, S, D, codes, 1, layout, power)
    slots = run_slots(runs)
    T = len(slots)
    size = torch.exp2(torch.randint(-12, 6, (T, Hk, 1), generator=g, device="cuda").float())
    kv = (torch.randn(2, T, Hk, D, generator=g, device="cuda") * size).to(dtype)
    k, v = kv[0], kv[1]
    f = -torch.rand(H, T, generator=g, device="cuda").t()
    want = reference_append(k, v, f, pages, slots, codes)
    versions = [t._version for t in pages]
    paged_append_8bit(k, v, f, *pages, torch.tensor(slots, device="cuda"))
    for name, a, b in zip(("k", "v", "k scales", "v scales", "gates"), pages, want):
        assert same(as_values(a), b), name
    assert all(t._version > n for t, n in zip(pages, versions))
    paged_append_8bit(k[:0], v[:0], f[:0], *pages, torch.zeros(0, dtype=torch.int64, device="cuda"))


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_append_of_every_value(codes, dtype):
    """All values of the type, NaN and infinities among them, in blocks of neighbouring magnitudes; a block of zeros, of NaN alone, of the smallest values."""
    from forgetting_transformer import paged_append_8bit
    D, S = 128, 16
    every = torch.arange(1 << 16, device="cuda", dtype=torch.int32).to(torch.int16).view(dtype)
    order = torch.argsort(torch.nan_to_num(every.float().abs(), nan=0.0), stable=True)
    mixed = every[torch.randperm(1 << 16, generator=torch.Generator(device="cuda").manual_seed(0), device="cuda")]
    rows = torch.cat([every[order].view(-1, 1, D), mixed.view(-1, 1, D), torch.zeros(S, 1, D, device="cuda", dtype=dtype), torch.full((S, 1, D), float("nan"), device="cuda", dtype=dtype)])
    T = len(rows)
    *pages, _ = pool(T // S, 1, 1, S, D, codes, 2)
    f = torch.zeros(T, 1, device="cuda")
    slots = list(range(T))
    want = reference_append(rows, rows.flip(0), f, pages, slots, codes)
    paged_append_8bit(rows, rows.flip(0).contiguous(), f, *pages, torch.arange(T, device="cuda"))
    for name, a, b in zip(("k", "v", "k scales", "v scales"), pages, want):
        assert same(as_values(a), b), name


def test_append_grows_a_block_token_by_token():
    """Sixteen tokens one at a time, ever larger, against the same rule applied to what is held."""
    from forgetting_transformer import paged_append_8bit
    for codes in CODES:
        *pages, g = pool(1, 2, 1, 32, 64, codes, 3)
        x = torch.randn(32, 1, 64, generator=g, device="cuda").bfloat16() * torch.exp2(torch.arange(32, device="cuda") * 0.5)[:, None, None].bfloat16()
        f = torch.zeros(32, 2, device="cuda")
        for t in range(32):
            want = reference_append(x[t:t + 1], -x[t:t + 1], f[t:t + 1], pages, [t], codes)
            paged_append_8bit(x[t:t + 1], -x[t:t + 1], f[t:t + 1], *pages, torch.tensor([t], device="cuda"))
            for a, b in zip(pages, want):
                assert same(as_values(a), b), (codes, t)
        # what is held is within half a step of every rounding on its way: at most twice the last one's
        G = 16
        for b in range(2):
            scale = pages[2][0, 0, b].double()
            off = (as_values(pages[0])[0, 0, G * b:G * b + G] * scale - x[G * b:G * b + G, 0].double()).abs()
            room = 2 * 0.5 * scale if codes == "int8" else x[G * b:G * b + G, 0].double().abs() * 2.0 ** -4 * 2 + scale * 2.0 ** -9
            assert (off <= room).all()


def ends_of(n):
    return torch.tensor([0] + n, dtype=torch.int32, device="cuda").cumsum(0, dtype=torch.int32)


def on_gpu(v, dtype=torch.int32):
    return torch.tensor(v, dtype=dtype, device="cuda")


@pytest.mark.parametrize("H,Hk,D,S,codes,dtype,lengths,pad,layout", [
    (1, 1, 16, 8, "e4m3", torch.bfloat16, [1], 0, "apart"), (6, 2, 32, 8, "int8", torch.float16, [0, 9, 64, 1, 0], 50, "between"),
    (12, 12, 64, 16, "int8", torch.float16, [33, 500, 16, 2], 3, "inside"), (16, 4, 128, 64, "e4m3", torch.bfloat16, [1000, 64, 0, 63], 700, "apart"),
    (4, 2, 64, 16, None, torch.bfloat16, [70, 5], 9, "apart"), (3, 3, 128, 32, None, torch.float16, [100, 0, 31], 1, "inside"),
    (5, 1, 32, 4096, "e4m3", torch.float16, [4097, 7], 0, "between"), (2, 2, 16, 16, "e4m3", torch.bfloat16, [(i * 7) % 40 for i in range(900)], 11, "apart")])
def test_gather(H, Hk, D, S, codes, dtype, lengths, pad, layout):
    from forgetting_transformer import paged_gather
    W = max(max(-(-n // S) for n in lengths), 1) + 1
    P = sum(-(-n // S) for n in lengths) + 2
    kp, vp, ks, vs, fp, g = pool(P, H, Hk, S, D, codes or "e4m3", 4, layout, power=False)
    scales = dict(k_scales=ks, v_scales=vs)
    if codes is None:
        kp, vp, scales = kp.float().to(dtype), vp.float().to(dtype), {}
    ids = torch.randperm(P, generator=torch.Generator().manual_seed(1)).tolist()
    table = [[ids.pop() for _ in range(-(-n // S))] for n in lengths]
    missing = [(b, i) for b, row in enumerate(table) for i in range(len(row)) if (b + i) % 11 == 10]
    for b, i in missing:
        table[b][i] = (-1, P, 2 ** 30)[i % 3]
    table = [row + [ids[0]] * (W - len(row)) for row in table]
    T = sum(lengths) + pad

    def check(got, who, n):
        at = 0
        for r, c in zip(who, n):
            pos = torch.arange(c, device="cuda")
            page = torch.tensor(table[r] if 0 <= r < len(table) else [-1] * W, device="cuda")[pos // S]
            here = ((page >= 0) & (page < P))[:, None]
            page, row = page.clamp(0, P - 1), pos % S
            for y, x, s in zip(got, (kp, vp, fp), (ks, vs, None)):
                w = x[page, :, row].float()
                if codes and s is not None:
                    w = w * s[page, :, row // min(S, 16)][..., None]
                w = torch.where(here if w.dim() == 2 else here[..., None], w, 0.0).to(y.dtype)
                assert torch.equal(y[at:at + c], w)
            at += c
        assert not any(y[at:].any() for y in got)

    got = paged_gather(kp, vp, fp, on_gpu(table), ends_of(lengths), max_tokens=T, dtype=dtype, **scales)
    assert [y.dtype for y in got] == [dtype, dtype, torch.float32] and got[0].shape == (T, Hk, D) and got[2].shape == (T, H)
    check(got, range(len(lengths)), lengths)
    who = [len(lengths) - 1, -1, 0, len(lengths) + 5, 0]
    n = [lengths[-1] // 2, 3, lengths[0], 2, lengths[0] // 2]
    check(paged_gather(kp, vp, fp, on_gpu(table), ends_of(n), max_tokens=sum(n) + 2, requests=on_gpu(who), dtype=dtype, **scales), who, n)
    assert [len(y) for y in paged_gather(kp, vp, fp, on_gpu(table), ends_of(lengths), max_tokens=0, dtype=dtype, **scales)] == [0, 0, 0]
    # ends beyond the places, beyond the table, that decrease or lie below zero: what is in range is read, nothing else
    for bad in ([0] + [2 ** 31 - 1] * len(lengths), [-5] * (len(lengths) + 1), [7] + [0] * len(lengths)):
        paged_gather(kp, vp, fp, on_gpu(table), on_gpu(bad), max_tokens=T, dtype=dtype, **scales)
    torch.cuda.synchronize()


def attention_reference(q, kp, vp, ks, vs, fp, table, lengths, requests, scale):
    P, Hk, S, D = kp.shape
    H = fp.shape[1]
    G = min(S, 16)
    out = torch.zeros_like(q, dtype=torch.float64)
    top = 0.0
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
        k, v = ((x[page, :, row].double() * s[page, :, row // G].double()[..., None]).transpose(0, 1).repeat_interleave(H // Hk, 0) for x, s in ((kp, ks), (vp, vs)))
        f = torch.where(here, fp[page, :, row].double().t(), 0.0)
        behind = torch.cat([f[:, 1:], f.new_zeros(H, 1)], -1).flip(-1).cumsum(-1).flip(-1)
        s = torch.where(here, (k * q[b].double()[:, None]).sum(-1) * scale + behind, float("-inf"))
        p = torch.softmax(s, -1)
        out[b] = torch.where((p > 0)[..., None], p[..., None] * v, 0.0).sum(1)
        top = max(top, v[:, here].abs().max().item())
    return out, top


def check_attention(got, want, top, dtype):
    bound = torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -12 * top
    err = (got.double() - want).abs()
    assert torch.isfinite(got).all()
    assert (err <= bound).all(), f"{(err / bound).max().item():.3f} of its bound"


def cache(P, H, Hk, S, D, codes, seed, layout="apart", power=False):
    """Pages as they are in earnest: values of size one."""
    kp, vp, ks, vs, f, g = pool(P, H, Hk, S, D, codes, seed, layout, power)
    for pages, scales in ((kp, ks), (vp, vs)):
        x = torch.randn(pages.shape, generator=g, device="cuda")
        G = min(S, 16)
        need = x.unflatten(2, (S // G, G)).abs().amax((-2, -1)) / CODES[codes][1]
        need = torch.exp2(need.log2().ceil()) if power else need * 1.1
        scales.copy_(need)
        y = (x.unflatten(2, (S // G, G)) / need[..., None, None]).flatten(2, 3)
        pages.copy_((y.round() if codes == "int8" else y).to(pages.dtype))
    return kp, vp, ks, vs, f, g


CASES = [  # B, H, Hk, D, S, W, lengths, codes, dtype, layout
    (1, 1, 1, 16, 8, 1, [1], "e4m3", torch.bfloat16, "apart"), (3, 2, 2, 32, 8, 4, [0, 1, 32], "int8", torch.float16, "between"),
    (4, 6, 3, 64, 16, 20, [5, 16, 17, 320], "e4m3", torch.bfloat16, "inside"), (2, 12, 12, 64, 16, 100, [1500, 1], "int8", torch.bfloat16, "apart"),
    (2, 8, 4, 128, 64, 40, [2560, 2499], "e4m3", torch.float16, "between"), (5, 4, 1, 16, 16, 200, [3200, 0, 7, 1024, 1025], "int8", torch.float16, "inside"),
    (5, 4, 1, 16, 16, 1200, [18000, 0, 7, 1024, 1025], "int8", torch.float16, "inside"), (3, 12, 4, 64, 32, 20, [0, 1, 640], "e4m3", torch.float16, "between"),
    (4, 20, 1, 128, 16, 30, [480, 33, 32, 257], "int8", torch.bfloat16, "apart"), (256, 1, 1, 128, 16, 20, None, "e4m3", torch.bfloat16, "inside"),
    (1, 40, 2, 128, 4096, 3, [9001], "e4m3", torch.bfloat16, "apart"), (70, 2, 1, 32, 32, 30, None, "e4m3", torch.bfloat16, "apart"),
    (130, 1, 1, 64, 8, 90, None, "int8", torch.float16, "between"), (1, 17, 1, 128, 32, 700, [22400], "int8", torch.bfloat16, "apart"),
    (6, 32, 2, 128, 256, 4, None, "e4m3", torch.bfloat16, "inside"), (300, 3, 3, 16, 8, 40, None, "e4m3", torch.float16, "apart"),
    (2, 16, 4, 32, 8, 3000, [24000, 200], "e4m3", torch.bfloat16, "apart"), (1100, 2, 2, 64, 16, 40, None, "int8", torch.bfloat16, "apart"),
    (256, 8, 1, 128, 16, 100, None, "e4m3", torch.float16, "apart")]


@pytest.mark.parametrize("B,H,Hk,D,S,W,lengths,codes,dtype,layout", CASES)
def test_attention(B, H, Hk, D, S, W, lengths, codes, dtype, layout):
    from forgetting_transformer import paged_forgetting_attention_8bit
    g = torch.Generator().manual_seed(B + W)
    if lengths is None:
        lengths = (torch.rand(B, generator=g) ** 3 * (W * S + 1)).long().tolist()
        lengths[0], lengths[-1] = 0, W * S
    P = sum(-(-n // S) for n in lengths) + 2
    kp, vp, ks, vs, fp, gen = cache(P, H, Hk, S, D, codes, 5, layout, power=B % 2 == 0)
    bad = float("nan") if codes == "e4m3" else -128
    kp[P - 1], vp[P - 1], ks[P - 1], vs[P - 1], fp[P - 1] = bad, bad, float("nan"), float("nan"), float("nan")        # a page that nobody holds
    ids = torch.randperm(P - 1, generator=g).tolist()
    table = [[ids.pop() for _ in range(-(-n // S))] for n in lengths]
    G = min(S, 16)
    for row, n in zip(table, lengths):             # what lies behind the last token of a page may be anything
        if n % S:
            kp[row[-1], :, n % S:], vp[row[-1], :, n % S:], fp[row[-1], :, n % S:] = bad, bad, float("nan")
            ks[row[-1], :, (n % S + G - 1) // G:], vs[row[-1], :, (n % S + G - 1) // G:] = float("inf"), float("nan")
    table = [row + [P - 1] * (W - len(row)) for row in table]
    q = torch.randn(B, H, D, generator=gen, device="cuda").to(dtype)
    args = (kp, vp, ks, vs, fp, on_gpu(table))
    out = paged_forgetting_attention_8bit(q, *args, on_gpu(lengths))
    assert out.dtype == dtype and out.shape == q.shape
    want, top = attention_reference(q, kp, vp, ks, vs, fp, table, lengths, None, D ** -0.5)
    check_attention(out, want, top, dtype)
    assert torch.equal(paged_forgetting_attention_8bit(q, *args, on_gpu(lengths)), out)
    if max(lengths) < W * S:
        check_attention(paged_forgetting_attention_8bit(q, *args, on_gpu(lengths), max_length=max(max(lengths), 1)), want, top, dtype)
    order = torch.randint(-1, B, (B + 3,), generator=g).tolist()                    # some requests twice, some rows without one
    seen = [lengths[r] // 2 + 1 if r >= 0 else 5 for r in order]
    seen = [min(n, lengths[r]) if r >= 0 else n for n, r in zip(seen, order)]
    q2 = torch.randn(B + 3, H, D, generator=gen, device="cuda").to(dtype)
    got = paged_forgetting_attention_8bit(q2, *args, on_gpu(seen), requests=on_gpu(order), sm_scale=0.3)
    check_attention(got, *attention_reference(q2, kp, vp, ks, vs, fp, table, seen, order, 0.3), dtype)


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_attention_pages_outside_the_pool_and_closed_gates(codes):
    from forgetting_transformer import paged_forgetting_attention_8bit
    B, H, Hk, D, S, W, P = 4, 6, 2, 64, 16, 40, 50
    kp, vp, ks, vs, fp, g = cache(P, H, Hk, S, D, codes, 6)
    table = torch.randint(0, P, (B, W), generator=torch.Generator().manual_seed(3)).tolist()
    table[0][3:7], table[1][W - 1], table[2] = [-1, P, 2 ** 30, -2 ** 31], -1, [-1] * W
    fp[table[3][10], :, 5], fp[table[3][30], 1, 15], fp[table[0][2], 2, 0] = -math.inf, -math.inf, -math.inf
    q = torch.randn(B, H, D, generator=g, device="cuda").bfloat16()
    lengths = [W * S, W * S - 3, 100, W * S]
    want, top = attention_reference(q, kp, vp, ks, vs, fp, table, lengths, None, D ** -0.5)
    check_attention(paged_forgetting_attention_8bit(q, kp, vp, ks, vs, fp, on_gpu(table), on_gpu(lengths)), want, top, torch.bfloat16)
    # lengths that no program of this library writes
    out = paged_forgetting_attention_8bit(q, kp, vp, ks, vs, fp, on_gpu(table), on_gpu([-3, 2 ** 31 - 1, 0, 5]))
    assert not out[0].any() and not out[2].any() and torch.isfinite(out).all()
    # gates that are not four in a row
    strided = torch.empty(P, S, H, device="cuda").transpose(1, 2).copy_(fp)
    check_attention(paged_forgetting_attention_8bit(q, kp, vp, ks, vs, strided, on_gpu(table), on_gpu(lengths)), want, top, torch.bfloat16)


@pytest.mark.parametrize("codes,dtype,H,Hk,D", [("e4m3", torch.bfloat16, 8, 2, 64), ("int8", torch.float16, 3, 3, 32)])
def test_a_run_of_all(codes, dtype, H, Hk, D):
    """Prompts in two pieces, then tokens one by one: slots, append, gather and packed attention for the prompts, attention over the pages for the tokens, against 64-bit attention
    over what the pages stand for."""
    from forgetting_transformer import forgetting_attention_packed, page_slots, paged_append_8bit, paged_forgetting_attention_8bit, paged_gather
    B, S, W, P = 5, 16, 20, 80
    g = torch.Generator(device="cuda").manual_seed(7)
    kp, vp, ks, vs, fp, _ = pool(P, H, Hk, S, D, codes, 8)
    lengths, table, free, count = on_gpu([0] * B), on_gpu([[-1] * W] * B), torch.arange(P, dtype=torch.int32, device="cuda"), on_gpu([P])
    u = torch.finfo(dtype).eps / 2

    def step(new, room):
        s = page_slots(lengths, on_gpu(new), table, free, count, page_size=S, max_tokens=room, in_place=True)
        x = [torch.randn(room, h, D, generator=g, device="cuda").to(dtype) for h in (H, Hk, Hk)]
        f = torch.nn.functional.logsigmoid(torch.randn(room, H, generator=g, device="cuda") + 2.0)
        paged_append_8bit(x[1], x[2], f, kp, vp, ks, vs, fp, s.slots)
        return s, x[0]

    for new in ([40, 0, 100, 7, 1], [13, 60, 1, 0, 33]):
        s, q = step(new, 200)
        cu_q, cu_k = ends_of(new), torch.cat([on_gpu([0]), lengths.cumsum(0, dtype=torch.int32)])
        total = int(lengths.sum())
        keys = paged_gather(kp, vp, fp, table, cu_k, max_tokens=total + 5, k_scales=ks, v_scales=vs, dtype=dtype)
        out = forgetting_attention_packed(q, *keys, cu_q, cu_k)
        at = 0
        for b, n in enumerate(new):
            seen = [int(lengths[b]) - n + i + 1 for i in range(n)]
            want, top = attention_reference(q[at:at + n], kp, vp, ks, vs, fp, table.tolist(), seen, [b] * n, D ** -0.5)
            # the gathered keys are rounded to 16 bits (exactly, the scales being powers of two); p is too, in the product with v
            assert ((out[at:at + n].double() - want).abs() <= u * want.abs() + (u + 2.0 ** -12) * top).all()
            at += n
        assert not out[at:].any()
    for _ in range(20):
        s, q = step([1, 1, 0, 1, 1], B)
        out = paged_forgetting_attention_8bit(q, kp, vp, ks, vs, fp, table, s.keys, requests=s.requests)
        want, top = attention_reference(q, kp, vp, ks, vs, fp, table.tolist(), s.keys.tolist(), s.requests.tolist(), D ** -0.5)
        check_attention(out, want, top, dtype)


def test_a_captured_step():
    """Slots, append and attention in one graph, replayed with the program's own work between, against the same steps in eager mode."""
    from forgetting_transformer import page_slots, paged_append_8bit, paged_forgetting_attention_8bit
    B, H, Hk, D, S, W, P = 4, 4, 2, 64, 16, 8, 40
    xs = [[torch.randn(B, h, D, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").bfloat16() for h in (H, Hk, Hk)] + [-torch.rand(B, H, device="cuda")] for i in range(30)]

    def fresh():
        kp, vp, ks, vs, fp, _ = pool(P, H, Hk, S, D, "e4m3", 9)
        return [kp, vp, ks, vs, fp, on_gpu([0] * B), on_gpu([[-1] * W] * B), torch.arange(P, dtype=torch.int32, device="cuda"), on_gpu([P])]

    def step(st, x, new):
        kp, vp, ks, vs, fp, lengths, table, free, count = st
        s = page_slots(lengths, new, table, free, count, page_size=S, max_tokens=B, in_place=True)
        paged_append_8bit(x[1], x[2], x[3], kp, vp, ks, vs, fp, s.slots)
        return paged_forgetting_attention_8bit(x[0], kp, vp, ks, vs, fp, table, s.keys, requests=s.requests)

    new, eager = on_gpu([1] * B), fresh()
    want = [step(eager, x, new) for x in xs]
    st, buf = fresh(), [t.clone() for t in xs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh(), buf, new)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(st, buf, new)
    for i, x in enumerate(xs):
        for b, t in zip(buf, x):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        step(eager, x, torch.zeros_like(new))
        torch.cuda.synchronize()


def test_refusals():
    from forgetting_transformer import paged_append_8bit, paged_forgetting_attention_8bit, paged_gather
    H, Hk, D, S, P, T = 4, 2, 64, 16, 6, 10
    kp, vp, ks, vs, fp, g = pool(P, H, Hk, S, D, "e4m3", 10)
    k, f, slots = torch.randn(T, Hk, D, device="cuda").bfloat16(), torch.zeros(T, H, device="cuda"), torch.arange(T, device="cuda")
    q, table, n = torch.randn(3, H, D, device="cuda").bfloat16(), on_gpu([[0, 1]] * 3), on_gpu([5, 6, 7])
    ok = dict(k=k, v=k, f=f, kp=kp, vp=vp, ks=ks, vs=vs, fp=fp, slots=slots)
    for bad in (dict(k=k.float()), dict(k=k[:, :1], v=k[:, :1]), dict(v=k.half()), dict(v=k[:-1]), dict(f=f[:, :2]), dict(f=f.double()), dict(slots=slots.int()), dict(slots=slots[:-1]),
                dict(kp=kp.view(torch.int8)), dict(kp=kp.view(torch.uint8), vp=vp.view(torch.uint8)), dict(ks=ks[:, :, :0]), dict(ks=ks.double()), dict(vs=vs[:-1]), dict(fp=fp[:, :3]),
                dict(kp=kp[..., :48], vp=vp[..., :48]), dict(kp=kp[..., 1:33], vp=vp[..., 1:33]), dict(fp=fp.half())):
        with pytest.raises(AssertionError):
            paged_append_8bit(*{**ok, **bad}.values())
    for bad in (dict(vp=kp), dict(vs=ks), dict(k=k.clone().requires_grad_()), dict(ks=vs, vs=vs)):
        with pytest.raises(RuntimeError):
            paged_append_8bit(*{**ok, **bad}.values())
    ok = dict(q=q, kp=kp, vp=vp, ks=ks, vs=vs, fp=fp, table=table, n=n)
    for bad in (dict(q=q[:, :2]), dict(q=q.float()), dict(table=table[:2]), dict(table=table.long()), dict(n=n[:2]), dict(n=n.long()), dict(ks=None)):
        with pytest.raises((AssertionError, AttributeError)):
            paged_forgetting_attention_8bit(*{**ok, **bad}.values())
    with pytest.raises(AssertionError):
        paged_forgetting_attention_8bit(*ok.values(), max_length=0)
    with pytest.raises(AssertionError):
        paged_forgetting_attention_8bit(*ok.values(), requests=on_gpu([0, 1]))
    cu = ends_of([5, 6, 7])
    sc = dict(k_scales=ks, v_scales=vs)
    for args, kw in (((kp, vp, fp, table, cu), dict(max_tokens=18)), ((kp, vp, fp, table, cu), dict(max_tokens=-1, **sc)), ((kp, vp, fp, table, cu), dict(max_tokens=18, dtype=torch.float32, **sc)),
                     ((kp, vp, fp, table, cu[:3]), dict(max_tokens=18, **sc)), ((kp, vp, fp, table, cu.long()), dict(max_tokens=18, **sc)),
                     ((kp.float().bfloat16(), vp.float().bfloat16(), fp, table, cu), dict(max_tokens=18, **sc)),
                     ((kp.float().bfloat16(), vp.float().bfloat16(), fp, table, cu), dict(max_tokens=18, dtype=torch.float16)), ((kp.float(), vp.float(), fp, table, cu), dict(max_tokens=18))):
        with pytest.raises(AssertionError):
            paged_gather(*args, **kw)


def test_what_the_kernels_do_not_take_is_copied():
    from forgetting_transformer import paged_append_8bit, paged_forgetting_attention_8bit
    H, Hk, D, S, P, T = 4, 2, 64, 16, 6, 40
    pages = list(pool(P, H, Hk, S, D, "int8", 11)[:5])
    other = [t.clone() for t in pages]
    wide = torch.randn(T, Hk, 2 * D + 1, device="cuda").bfloat16()[..., 1:D + 1]
    f = -torch.rand(T, H, device="cuda")
    slots = torch.arange(3, T + 3, device="cuda")
    paged_append_8bit(wide, wide, f, *pages, torch.stack([slots, slots], 1)[:, 0])
    paged_append_8bit(wide.contiguous(), wide.contiguous(), f, *other, slots)
    assert all(torch.equal(a.view(torch.uint8) if a.dtype == torch.int8 else a, b.view(torch.uint8) if b.dtype == torch.int8 else b) for a, b in zip(pages, other))
    q = torch.randn(2, H, D + 3, device="cuda").half()[..., 3:]
    table, n = on_gpu([[0, 1, 2], [3, 4, 5]]), on_gpu([40, 17])
    a = paged_forgetting_attention_8bit(q, *pages, table.t().contiguous().t(), torch.stack([n, n], 1)[:, 0])
    assert torch.equal(a, paged_forgetting_attention_8bit(q.contiguous(), *pages, table, n))


@pytest.mark.parametrize("codes,dtype,H,Hk", [("e4m3", torch.bfloat16, 6, 2), ("int8", torch.float16, 4, 4), (None, torch.bfloat16, 3, 3)])
def test_cache_of_a_model(codes, dtype, H, Hk):
    """PagedFgateCache over two layers: prompts in pieces, refused and idle requests, tokens, a release; against attention over everything that each request has brought."""
    from forgetting_transformer import PagedFgateCache
    D, B, S, layers = 64, 4, 16, 2
    cache_ = PagedFgateCache(layers, H, D, num_pages=24, max_requests=B, max_length=200, page_size=S, dtype=dtype, cache_dtype=CODES[codes][0] if codes else None, num_kv_heads=Hk)
    g = torch.Generator(device="cuda").manual_seed(12)
    u = torch.finfo(dtype).eps / 2

    def held(layer):
        ks, vs = (x[layer] if x is not None else torch.ones(24, Hk, 1, device="cuda") for x in (cache_.key_scales, cache_.value_scales))
        return cache_.key_pages[layer], cache_.value_pages[layer], ks, vs, cache_.log_fgate_pages[layer]

    def step(new, room, prompts, max_keys=None):
        s = cache_.schedule(on_gpu(new), room, prompts=prompts)
        for layer in range(layers):
            q, k, v = (torch.randn(room, h, D, generator=g, device="cuda").to(dtype) for h in (H, Hk, Hk))
            cache_.update(k, v, torch.nn.functional.logsigmoid(torch.randn(room, H, generator=g, device="cuda") + 2.0), layer)
            out = cache_.attend_prompts(q, layer, max_keys=max_keys) if prompts else cache_.attend(q, layer)
            kp, vp, ks, vs, fp = held(layer)
            if codes is None:      # the reference takes a block of sixteen tokens
                ks, vs = (x.expand(24, Hk, S // 16).contiguous() for x in (ks, vs))
            want, top = attention_reference(q, kp, vp, ks, vs, fp, cache_.block_table.tolist(), s.keys.tolist(), s.requests.tolist(), D ** -0.5)
            assert ((out.double() - want).abs() <= u * want.abs() + ((u if prompts else 0.0) + 2.0 ** -12) * top).all()
            assert not out[s.requests < 0].any()
        return s

    step([50, 0, 90, 17], 200, True)
    s = step([30, 5, 0, 300], 400, True)          # the last one has no room
    assert s.granted.tolist()[3] is False
    step([1, 1, 1, 1], B, False)
    step([1, 0, 1, 0], B, True, max_keys=400)
    cache_.release(on_gpu([True, False, False, False], torch.bool))
    step([40, 3, 3, 3], 60, True)
    step([1, 1, 1, 1], B, False)


def test_a_captured_step_of_prompts():
    """The cache's step of prompts in a graph, replayed for pieces of other lengths with eager work between."""
    from forgetting_transformer import PagedFgateCache
    H, D, B, room = 4, 32, 3, 64
    make = lambda: PagedFgateCache(1, H, D, num_pages=30, max_requests=B, max_length=160, page_size=16, cache_dtype=torch.float8_e4m3fn)
    gen = torch.Generator(device="cuda").manual_seed(13)
    xs = [[torch.randn(room, H, D, generator=gen, device="cuda").bfloat16() for _ in range(3)] + [-torch.rand(room, H, generator=gen, device="cuda"), on_gpu(n)]
          for n in ([20, 1, 0], [5, 30, 29], [0, 0, 3], [40, 2, 2], [1, 1, 1])]

    def step(cache_, x):
        cache_.schedule(x[4], room, prompts=True)
        cache_.update(x[1], x[2], x[3], 0)
        return cache_.attend_prompts(x[0], 0)

    eager = make()
    want = [step(eager, x) for x in xs]
    cache_, buf = make(), [t.clone() for t in xs[0]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(make(), buf)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(cache_, buf)
    for i, x in enumerate(xs):
        for b, t in zip(buf, x):
            b.copy_(t)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        step(eager, [*x[:4], torch.zeros_like(x[4])])
        torch.cuda.synchronize()


@pytest.mark.parametrize("codes", ["e4m3", "int8"])
def test_a_pool_of_more_than_four_gibibytes(codes):
    """Pages whose codes lie behind 2**32: the same bits as from a small pool, for the append, the gather and the attention."""
    from forgetting_transformer import paged_append_8bit, paged_forgetting_attention_8bit, paged_gather
    S, Hk, H, D, n = 128, 4, 8, 128, 300
    far = (1 << 32) // (S * Hk * D)
    g = torch.Generator(device="cuda").manual_seed(14)
    k, v = (torch.randn(n, Hk, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    f, q = -torch.rand(n, H, generator=g, device="cuda"), torch.randn(1, H, D, generator=g, device="cuda").bfloat16()
    got = []
    for first, P in ((0, 3), (far, far + 3)):
        empty = lambda *s, t=CODES[codes][0]: torch.empty(s, dtype=t, device="cuda")
        kp, vp, fp = empty(P, Hk, S, D), empty(P, Hk, S, D), empty(P, H, S, t=torch.float32)
        ks, vs = empty(P, Hk, S // 16, t=torch.float32), empty(P, Hk, S // 16, t=torch.float32)
        pages = [first + 2, first, first + 1]
        slots = torch.tensor([p * S + i for p in pages for i in range(S)], device="cuda")[:n].contiguous()
        paged_append_8bit(k, v, f, kp, vp, ks, vs, fp, slots)
        table, wide = on_gpu([pages]), on_gpu([pages + [-1] * 60])        # (a row whole, and in pieces)
        out = paged_gather(kp, vp, fp, table, on_gpu([0, n]), max_tokens=n, k_scales=ks, v_scales=vs)
        got.append([*out, *(paged_forgetting_attention_8bit(q, kp, vp, ks, vs, fp, t, on_gpu([m])) for t, m in ((table, n), (table, 17), (wide, n)))])
        del kp, vp
    assert all(torch.isfinite(a).all() and torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("which", ["pages", "heads", "tokens", "scales"])
def test_append_refuses_pages_that_lie_on_each_other(which):
    """Keys and values that share memory without beginning at one place; the same pools taken apart are written as separate ones are."""
    from forgetting_transformer import paged_append_8bit
    H, Hk, D, S, P, T = 4, 2, 64, 16, 6, 40
    g = torch.Generator(device="cuda").manual_seed(15)
    k, v = (torch.randn(T, Hk, D, generator=g, device="cuda").bfloat16() for _ in range(2))
    f, slots = -torch.rand(T, H, generator=g, device="cuda"), torch.arange(T, device="cuda")
    zeros = lambda *s, t=torch.int8: torch.zeros(s, dtype=t, device="cuda")
    pages, scales, fp = [zeros(P, Hk, S, D) for _ in range(2)], [zeros(P, Hk, 1, t=torch.float32) for _ in range(2)], zeros(P, H, S, t=torch.float32)
    bad_pages, bad_scales = pages, scales
    if which == "pages":
        x = zeros(P + 1, Hk, S, D)
        bad_pages = [x[:-1], x[1:]]
    elif which == "heads":
        x = zeros(P, Hk + 1, S, D)
        bad_pages = [x[:, 1:], x[:, :-1]]
    elif which == "tokens":
        x = zeros(P, S + 2, Hk, D).transpose(1, 2)
        bad_pages = [x[:, :, :S], x[:, :, 2:]]
    else:
        x = zeros(P + 3, Hk, 1, t=torch.float32)
        bad_scales = [x[:-3], x[3:]]
    with pytest.raises(RuntimeError, match="may not overlap"):
        paged_append_8bit(k, v, f, *bad_pages, *bad_scales, fp, slots)
    paged_append_8bit(k, v, f, *pages, *scales, fp, slots)
    kv, sc = zeros(P, Hk, 2, S, D), zeros(P, 2, Hk, 1, t=torch.float32)
    between = [kv[:, :, 0], kv[:, :, 1], sc[:, 0], sc[:, 1], torch.zeros_like(fp)]
    paged_append_8bit(k, v, f, *between, slots)
    assert all(torch.equal(a, b) for a, b in zip(between, (*pages, *scales, fp)))


def prompts_cache(lengths, codes=None, **more):
    """A cache of one layer whose requests have just brought `lengths` tokens, and the step's queries."""
    from forgetting_transformer import PagedFgateCache
    H, D, B = 4, 64, len(lengths)
    c = PagedFgateCache(1, H, D, **{**dict(num_pages=40, max_requests=B, max_length=160, page_size=16, cache_dtype=CODES[codes][0] if codes else None), **more})
    g = torch.Generator(device="cuda").manual_seed(16)
    room = sum(lengths) + 5
    q, k, v = (torch.randn(room, H, D, generator=g, device="cuda").bfloat16() for _ in range(3))
    f = torch.nn.functional.logsigmoid(torch.randn(room, H, generator=g, device="cuda") + 2.0)

    def step(new=None):
        c.schedule(on_gpu(lengths) if new is None else new, room, prompts=True)
        c.update(k, v, f, 0)
    return c, q, step


@pytest.mark.parametrize("codes", ["int8", None])
def test_prompts_past_max_keys_give_zeros(codes):
    """A request whose keys do not fit gives zeros, and so do those behind it; the ones in front are whole."""
    lengths = [50, 0, 60, 70, 33]
    c, q, step = prompts_cache(lengths, codes)
    step()
    ks, vs = (x[0] if x is not None else torch.ones(40, 4, 1, device="cuda") for x in (c.key_scales, c.value_scales))
    s = c.step
    want, top = attention_reference(q, c.key_pages[0], c.value_pages[0], ks, vs, c.log_fgate_pages[0], c.block_table.tolist(), s.keys.tolist(), s.requests.tolist(), 64 ** -0.5)
    u = 2.0 ** -8
    for max_keys, fits in ((213, 213), (212, 180), (500, 213), (109, 50), (110, 110), (179, 110), (50, 50), (49, 0), (1, 0)):
        out = c.attend_prompts(q, 0, max_keys=max_keys)
        assert ((out[:fits].double() - want[:fits]).abs() <= u * want[:fits].abs() + (u + 2.0 ** -12) * top).all(), max_keys
        assert not out[fits:].any(), max_keys


def test_a_captured_step_of_prompts_with_max_keys():
    """The same in a graph, replayed for pieces of other lengths with eager work between; some of them do not fit."""
    xs = [on_gpu(n) for n in ([20, 1, 0], [5, 30, 29], [0, 0, 3], [40, 2, 2], [1, 1, 1])]
    make = lambda: prompts_cache([20, 40, 40], "e4m3")
    eager, q, step = make()
    want = []
    for new in xs:
        step(new)
        want.append(eager.attend_prompts(q, 0, max_keys=75))
    assert want[1][:35].any() and not want[1][35:].any() and want[3][:40].any() and not want[3][40:].any()
    c, q, step = make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other, _, warm = make()
        warm(xs[0])
        other.attend_prompts(q, 0, max_keys=75)
    torch.cuda.current_stream().wait_stream(side)
    new, graph = xs[0].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(new)
        out = c.attend_prompts(q, 0, max_keys=75)
    for i, x in enumerate(xs):
        new.copy_(x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i]), i
        eager.attend_prompts(q, 0, max_keys=60)
        torch.cuda.synchronize()


def test_room_of_prompts_without_max_keys():
    """No more than the step's requests can hold, where the pool is larger."""
    c, q, step = prompts_cache([50, 60], "e4m3", num_pages=1 << 16, max_length=64)
    step()
    want = c.attend_prompts(q, 0, max_keys=128)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    out = c.attend_prompts(q, 0)
    assert torch.equal(out, want)
    keys = 2 * 64                                       # of k, v, gates, their sums; of the queries o; plan and parts as they come
    assert torch.cuda.max_memory_allocated() - before <= keys * 4 * (2 * 64 * 2 + 4 + 8) + q.numel() * 2 + (8 << 20)
    few = q[:1].contiguous()
    c.schedule(on_gpu([0, 1]), 1, prompts=True)
    c.update(few, few, torch.zeros(1, 4, device="cuda"), 0)
    assert torch.equal(c.attend_prompts(few, 0), c.attend_prompts(few, 0, max_keys=64))
