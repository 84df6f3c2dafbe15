"""Attention over pages with gates that keep every key alive, so that each piece, wave, batch and window of the block table has a visible share of the result.

The values are marks: every unit of keys (a page, or the keys that a wave loads at once where those are fewer) has 1 in one element of the head and 0 in the others, so an
element of the output is the share of the softmax that its units have together.  Nothing cancels, so the tolerance is relative: half a step of the output's type
and 2^-13 for 32-bit arithmetic (a score is off by at most 13 roundings of |q||k| scale log2(e) < 16 and a few of its gates, below 2^-16; numerator and denominator are sums
with chains of fewer than 1024 links, 2^-14 each; the hardware's exponential adds 2^-22).  Whether that would notice a lost unit is tested as well, with the mistakes planted in the
reference."""
import pytest
import torch

CASES = [  # H, D, S, lengths, dtype, heads inside: one row of a request each
    (1, 128, 32, [22400], torch.bfloat16, False), (2, 128, 4096, [9001, 5000], torch.float16, True), (2, 64, 16, [1500, 64, 9600], torch.bfloat16, True),
    (1, 64, 8, [7001], torch.float16, False), (2, 32, 8, [9003, 300], torch.float16, False), (2, 32, 32, [24000, 300], torch.bfloat16, False), (2, 16, 16, [3200, 24013, 0, 1025], torch.float16, False),
    (16, 128, 16, [2047] * 6, torch.bfloat16, False), (3, 16, 64, [9000, 1] * 3, torch.bfloat16, True)]
PLANNED = [  # the same with so many rows that their plan is made in front
    (2, 32, 16, [6000, 5001, 3333] * 100, torch.bfloat16, False), (1, 128, 64, [3000, 100] * 128, torch.float16, True), (2, 64, 16, [2600] * 256 + [12000], torch.bfloat16, False)]


def make(H, D, S, lengths, dtype, inside, device):
    """Queries, pages and the block table, and each key's unit and each unit's element of the head."""
    g = torch.Generator(device=device).manual_seed(sum(lengths) + D)
    rnd = lambda *s: torch.randn(*s, generator=g, device=device)
    counts = [-(-n // S) for n in lengths]
    P, W = sum(counts) + 1, max(counts) + 1
    order = torch.randperm(P, generator=g, device=device)
    shape = lambda *tail: (P, S, H, *tail) if inside else (P, H, S, *tail)
    turn = lambda t: t.transpose(1, 2) if inside else t
    kp, vp, fp = turn(rnd(*shape(D)).to(dtype)), turn(torch.full(shape(D), 3.0, dtype=dtype, device=device)), turn(torch.full(shape(), -3.0, device=device))
    q = rnd(len(lengths), H, D).to(dtype)
    table = torch.full((len(lengths), W), int(order[-1]), dtype=torch.int32, device=device)      # a page of wrong values behind every request's last
    unit, at, rows = min(S, 4096 // D), 0, []
    for b, (n, c) in enumerate(zip(lengths, counts)):
        ids = order[at:at + c]
        table[b, :c] = ids.int()
        at += c
        marks = torch.randint(0, D, (-(-c * S // unit),), generator=g, device=device)
        element = marks[torch.arange(c * S, device=device) // unit]
        f = -2.0 / max(n, 1) * torch.rand(H, c * S, generator=g, device=device)
        f[:, torch.randint(0, max(c * S, 1), (3,), generator=g, device=device) if c else []] = -0.25     # steps that every piece in front has to hear of
        vp[ids] = torch.nn.functional.one_hot(element, D).to(dtype).view(c, 1, S, D).expand(c, H, S, D)
        fp[ids] = f.view(H, c, S).transpose(0, 1)
        rows.append((ids, marks, element))
    return q, kp, vp, fp, table, unit, rows


def shares(q, kp, fp, ids, n, scale, shifted=True):
    """(H, n): what each key weighs in the softmax; without ``shifted`` the gates are forgotten."""
    k, f = (t[ids].double().transpose(0, 1).flatten(1, 2)[:, :n] for t in (kp, fp))
    behind = f.sum(-1, keepdim=True) - f.cumsum(-1)
    return torch.softmax((k * q.double()[:, None]).sum(-1) * scale + (behind if shifted else 0.0), -1)


def by_element(p, element, D):
    return torch.zeros(p.shape[0], D, dtype=p.dtype, device=p.device).index_add_(1, element[:p.shape[1]], p)


def bound(want, dtype):
    return (torch.finfo(dtype).eps / 2 + 2.0 ** -13) * want + (2.0 ** -25 if dtype == torch.float16 else 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(CASES) + len(PLANNED)))
def test_every_key_has_its_share(case):
    from forgetting_transformer import paged_forgetting_attention
    H, D, S, lengths, dtype, inside = (CASES + PLANNED)[case]
    q, kp, vp, fp, table, _, rows = make(H, D, S, lengths, dtype, inside, "cuda")
    n = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = paged_forgetting_attention(q, kp, vp, fp, table, n)
    back = torch.arange(len(lengths) - 1, -1, -1, dtype=torch.int32, device="cuda")             # rows in another order than the table's
    again = paged_forgetting_attention(q.flip(0), kp, vp, fp, table, n.flip(0), requests=back).flip(0)
    for b, (ids, _, element) in enumerate(rows):
        if lengths[b] == 0:
            assert out[b].abs().max() == 0 and again[b].abs().max() == 0
            continue
        want = by_element(shares(q[b], kp, fp, ids, lengths[b], D ** -0.5), element, D)
        for got in (out[b], again[b]):
            err = (got.double() - want).abs()
            assert (err <= bound(want, dtype)).all(), f"row {b}: {(err / bound(want, dtype)).max().item():.2f} of its bound"


@pytest.mark.parametrize("case", range(len(CASES)))
def test_the_tolerance_notices_what_is_lost(case):
    """Each unit dropped, pages of the next window read, pieces and waves left out, gates of the pieces behind forgotten: none stays inside the tolerance."""
    H, D, S, lengths, dtype, inside = CASES[case]
    q, kp, vp, fp, table, unit, rows = make(H, D, S, lengths, dtype, inside, "cpu")
    for b, (ids, marks, element) in enumerate(rows):
        n = lengths[b]
        if n < 2 * unit:
            continue
        p = shares(q[b], kp, fp, ids, n, D ** -0.5)
        want = by_element(p, element, D)
        allowed = bound(want, dtype)

        def noticed(wrong):
            return ((wrong - want).abs() > allowed).any(-1)

        of_unit = torch.zeros(H, len(marks), dtype=torch.float64).index_add_(1, torch.arange(n) // unit, p)
        for u in range(-(-n // unit)):                                         # a lost unit: its element gives up the share, the others grow
            wrong = want.clone()
            wrong[:, marks[u]] -= of_unit[:, u]
            assert noticed(wrong / (1.0 - of_unit[:, u:u + 1])).all(), f"unit {u} of row {b}"
        batch = 16384 // D
        masks = []
        if n > batch:
            masks.append(torch.arange(n) >= n - batch)                         # only the last batch
            masks.append((n - 1 - torch.arange(n)) % batch < batch // 4 * 3)   # a wave of each batch left out
        for keep in masks:
            kept = p * keep
            assert noticed(by_element(kept / kept.sum(-1, keepdim=True), element, D)).all()
        if n > 64 * S:                                                         # a window of the table one late: the keys of its last 64 pages twice
            late = torch.cat([ids[:64], ids[:len(ids) - 64]])
            wrong = shares(q[b], kp, fp, late, n, D ** -0.5)
            shown = torch.cat([element[:64 * S], element[:len(element) - 64 * S]])
            assert noticed(by_element(wrong, shown, D)).all()
        assert noticed(by_element(shares(q[b], kp, fp, ids, n, D ** -0.5, shifted=False), element, D)).all()
