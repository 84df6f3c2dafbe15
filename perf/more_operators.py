"""Forgetting Attention over packed sequences, and serving it from pages that hold keys and values in 8 bits, as timed cases with their plain forms.

A case is a dict of plain values.  ``op`` names the operator:

  packed    ``forgetting_attention_packed``: B sequences of up to ``longest`` tokens one after the other, H query heads on Hk key heads, behind ``pad`` places
            that belong to nobody; with ``prefix`` every sequence also sees up to so many tokens in front of its own; with ``grad`` forward and backward
  append    ``paged_append_8bit``: T new tokens into their slots, one each for T requests or the prompts of ``requests`` of them; ``skipped`` have no slot
  gather    ``paged_gather``: the cached tokens of B requests, one request after the other, as 16-bit keys and values
  attend    ``paged_forgetting_attention_8bit``: one new token for each of B requests that hold between ``shortest`` and ``longest`` tokens

Pages hold 8-bit keys and values, in e4m3 or in whole numbers, with a scale for every block of 16 tokens (8 on pages of 8) and head.

``draw_seed`` fixes what the amount of work depends on (how long each sequence is); everything else comes from the seed of ``prepare``.
"""
import math
import random
import sys
from pathlib import Path

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_CODES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
_LARGEST = {"e4m3": 448.0, "int8": 127.0}


def _ft():
    pkg = str(Path.cwd() / "forgetting-transformer_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import forgetting_transformer
    return forgetting_transformer


def _packed(name, B, H, Hk, D, shortest, longest, *, prefix=0, pad=0, dtype="bf16", grad=False, draw_seed=0):
    return dict(name=name, op="packed", B=B, H=H, Hk=Hk, D=D, shortest=shortest, longest=longest, prefix=prefix, pad=pad, dtype=dtype, grad=grad, draw_seed=draw_seed)


def _append(name, T, requests, H, Hk, D, page, *, codes="e4m3", dtype="bf16", skipped=0, draw_seed=0):
    return dict(name=name, op="append", T=T, requests=requests, H=H, Hk=Hk, D=D, page=page, codes=codes, dtype=dtype, skipped=skipped, draw_seed=draw_seed)


def _gather(name, B, H, Hk, D, page, shortest, longest, *, pad=0, codes="e4m3", dtype="bf16", draw_seed=0):
    return dict(name=name, op="gather", B=B, H=H, Hk=Hk, D=D, page=page, shortest=shortest, longest=longest, pad=pad, codes=codes, dtype=dtype, draw_seed=draw_seed)


def _attend(name, B, H, Hk, D, page, shortest, longest, *, codes="e4m3", dtype="bf16", draw_seed=0):
    return dict(_gather(name, B, H, Hk, D, page, shortest, longest, codes=codes, dtype=dtype, draw_seed=draw_seed), op="attend")


def listed():
    return [
        # one step of a few requests whose prompts come in pieces, next to one that is at its last token
        _packed("packed_chunk", 6, 12, 12, 64, 1, 64, prefix=900, pad=16, dtype="fp16", draw_seed=1),
        # the prompts of one step, of very different lengths, in a step with room for more tokens
        _packed("packed_prompts", 24, 16, 4, 128, 20, 2048, pad=512, draw_seed=2),
        # pieces of long prompts whose beginning is cached
        _packed("packed_far", 4, 16, 4, 128, 200, 1024, prefix=12288, draw_seed=3),
        # a training step on documents packed into one row
        _packed("packed_step", 8, 12, 12, 64, 128, 2048, grad=True, draw_seed=4),
        # long documents, four query heads on a key head
        _packed("packed_long", 8, 16, 4, 128, 1500, 4096, grad=True, draw_seed=5),
        # the next tokens of 48 requests into the pages of one layer
        _append("append8_tokens", 48, 48, 12, 12, 64, 16, codes="int8", dtype="fp16", draw_seed=6),
        # prompts into the pages of one layer, some tokens refused
        _append("append8_prompts", 16384, 20, 16, 4, 128, 64, skipped=100, draw_seed=7),
        # what a few requests have cached, for the next piece of their prompts
        _gather("gather8_prefixes", 6, 12, 12, 64, 16, 0, 900, pad=70, codes="int8", dtype="fp16", draw_seed=8),
        # the same for long ones
        _gather("gather8_long", 8, 16, 4, 128, 64, 6000, 12288, draw_seed=9),
        # a single user generates from a short cache
        _attend("attend8_single", 1, 12, 12, 64, 16, 1500, 1500, draw_seed=10),
        # 48 requests of very different lengths, some of them idle
        _attend("attend8_ragged", 48, 12, 12, 64, 16, 0, 8192, codes="int8", dtype="fp16", draw_seed=11),
        # a large batch generates from long caches, four query heads on a key head
        _attend("attend8_long", 32, 16, 4, 128, 64, 24576, 32768, draw_seed=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


_MAX_SCORES = 8 * 16 * 4096 * 4096       # of packed_long, with the shorter sequences filled up
_MAX_TOKENS = 16384 * 4 * 128            # elements of the keys of append8_prompts
_MAX_CACHE = 32 * 4 * 32768 * 128        # elements of the keys of attend8_long
_HEADS = [1, 2, 3, 5, 8, 12, 12, 16, 16, 32]


def draw(rng):
    op = rng.choice(["packed", "packed", "packed", "append", "gather", "attend", "attend"])
    D = rng.choice([16, 32, 64, 64, 128, 128])
    H, dtype, codes = rng.choice(_HEADS), rng.choice(["bf16", "bf16", "fp16"]), rng.choice(["e4m3", "e4m3", "int8"])
    Hk = rng.choice([h for h in range(1, H + 1) if H % h == 0])
    page, draw_seed = rng.choice([8, 16, 16, 32, 64, 128]), rng.randrange(1 << 20)
    if op == "packed":
        longest = _log_int(rng, 1, 8192)
        shortest, prefix = rng.choice([0, 1, longest // 2, longest]), rng.choice([0, 0, 0, _log_int(rng, 1, 16384)])
        B = _log_int(rng, 1, 64)
        while B > 1 and B * H * longest * (longest + prefix) > _MAX_SCORES:
            B -= 1
        while B * H * longest * (longest + prefix) > _MAX_SCORES:
            prefix //= 2
            longest = max(longest * 3 // 4, 1)
        grad = longest > 1 and rng.random() < 0.5
        case = _packed("", B, H, Hk, D, min(shortest, longest), longest, prefix=prefix, pad=rng.choice([0, 0, rng.randrange(1, 600)]), dtype=dtype, grad=grad, draw_seed=draw_seed)
    elif op == "append":
        T = _log_int(rng, 1, 16384)
        while T * Hk * D > _MAX_TOKENS:
            T = T // 2 + 1
        requests = T if rng.random() < 0.5 and T <= 1024 else _log_int(rng, 1, min(T, 64))
        case = _append("", T, requests, H, Hk, D, page, codes=codes, dtype=dtype, skipped=rng.choice([0, 0, T // 5]), draw_seed=draw_seed)
    else:
        longest = _log_int(rng, 16, 32768 if op == "attend" else 16384)
        shortest = rng.choice([0, 1, longest // 2, longest])
        B = _log_int(rng, 1, 64)
        while B > 1 and B * Hk * longest * D > (_MAX_CACHE if op == "attend" else 8 * _MAX_TOKENS) or B * H * longest * 2 > _MAX_CACHE // 16:
            B, longest = max(B - 1, 1), longest if B > 1 else longest // 2
        shortest = min(shortest, longest)
        args = dict(codes=codes, dtype=dtype, draw_seed=draw_seed)
        if op == "gather":
            case = _gather("", B, H, Hk, D, page, shortest, longest, pad=rng.choice([0, rng.randrange(1, 300)]), **args)
        else:
            case = _attend("", B, H, Hk, D, page, shortest, longest, **args)
    del case["name"]
    return case


def _spread(rng, count, lo, hi):
    """`count` lengths over the logarithm from the shortest to the longest, some of them 0 where that is the shortest; one is the longest."""
    n = [min(hi, max(lo, _log_int(rng, max(lo, 1), max(hi, 1)) if lo or rng.random() > 0.1 else 0)) for _ in range(count)]
    n[rng.randrange(count)] = hi
    return n


def _sequences(case):
    """New tokens of each sequence, and the tokens in front of them."""
    rng = random.Random(case["draw_seed"])
    new = _spread(rng, case["B"], case["shortest"], case["longest"])
    return new, _spread(rng, case["B"], 0, case["prefix"]) if case["prefix"] else [0] * case["B"]


def _lengths(case):
    """Cached tokens of each request."""
    return _spread(random.Random(case["draw_seed"]), case["B"], case["shortest"], case["longest"])


def _runs(case):
    """New tokens of each request of an append, and how many it has in front of them on the page that they start on."""
    rng = random.Random(case["draw_seed"])
    R, T, S = case["requests"], case["T"], case["page"]
    if R == T:
        n = [1] * T
    else:
        cuts = sorted(rng.sample(range(1, T), R - 1))
        n = [b - a for a, b in zip([0] + cuts, cuts + [T])]
    return n, [rng.randrange(S) if R == T or rng.random() < 0.5 else 0 for _ in n]


def _block(page):
    return min(page, 16)


def _scale_of(amax, codes):
    """The smallest power of two by which a block with this largest magnitude fits its codes."""
    m, e = torch.frexp(amax / _LARGEST[codes])                 # amax / largest = m 2^e, m in [1/2, 1)
    e = torch.where(m == 0.5, e - 1, e).clamp(min=-126)
    return ((torch.where(amax > 0, e, -126) + 127).int() << 23).view(torch.float32)


def _coded(x, codes):
    """The nearest codes of values that are divided by their scale (ties to the even one)."""
    x = x.clamp(-_LARGEST[codes], _LARGEST[codes])
    return (x.round() if codes == "int8" else x).to(_CODES[codes])


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, H, Hk, D = case["op"], case["H"], case["Hk"], case["D"]
    dt = _DTYPES[case["dtype"]]
    st = dict(case=case)

    def rnd(*shape, dtype=torch.float32):
        return torch.randn(*shape, generator=gen, device=dev, dtype=dtype)

    def ends(n):
        return torch.tensor([0] + n, dtype=torch.int32, device=dev).cumsum(0, dtype=torch.int32)

    def gates(*shape):
        return torch.nn.functional.logsigmoid(rnd(*shape) + 3.0)

    if op == "packed":
        new, front = _sequences(case)
        T, N = sum(new) + case["pad"], sum(new) + sum(front) + case["pad"]
        st.update(cu_seqlens=ends(new), q=rnd(T, H, D, dtype=dt), k=rnd(N, Hk, D, dtype=dt), v=rnd(N, Hk, D, dtype=dt), log_fgate=gates(N, H))
        st["cu_seqlens_k"] = ends([a + b for a, b in zip(new, front)]) if case["prefix"] else None
        if case["grad"]:
            st["leaves"] = [st[n].requires_grad_() for n in ("q", "k", "v", "log_fgate")]
            st["dout"] = rnd(T, H, D, dtype=dt)
        return st

    S, codes = case["page"], case["codes"]
    if op == "append":
        new, at = _runs(case)
        lens = [a + n for a, n in zip(at, new)]
    else:
        lens = _lengths(case)
    counts = [(n + S - 1) // S for n in lens]
    width, pool = max(max(counts), 1), sum(counts) + 3
    ids = torch.randperm(pool, generator=gen, device=dev)[:sum(counts)]
    # the pages of a request follow each other in `ids`, and so do the requests
    first = ends(counts)[:-1, None].long()
    cols = torch.arange(width, device=dev)
    used = cols < torch.tensor(counts, device=dev)[:, None]
    table = torch.where(used, torch.cat([ids, ids.new_zeros(1)])[(first + cols).clamp(max=len(ids))], 0).int()
    # cached keys and values: every head has a size of its own, as projections and norms leave them
    G = _block(S)
    for n in ("k", "v"):
        x = rnd(pool, Hk, S // G, G, D) * (0.6 * rnd(Hk, 1, 1, 1)).exp()
        scale = _scale_of(x.abs().amax((-2, -1)), codes)
        st[n + "_scales"] = scale
        st[n + "_pages"] = _coded(x / scale[..., None, None], codes).view(pool, Hk, S, D)
        del x
    st["log_fgate_pages"] = gates(pool, H, S)
    if op == "append":
        T = case["T"]
        size = (0.6 * rnd(Hk, 1)).exp()
        st.update(k=(rnd(T, Hk, D) * size).to(dt), v=(rnd(T, Hk, D) * size).to(dt), log_fgate=gates(T, H))
        who = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
        pos = torch.arange(T, device=dev) - ends(new)[:-1][who] + torch.tensor(at, device=dev)[who]
        slots = table[who, pos // S].long() * S + pos % S
        if case["skipped"]:       # the last tokens found no room
            slots[T - case["skipped"]:] = -1
        st["slots"] = slots
    elif op == "gather":
        st.update(block_table=table, cu_seqlens=ends(lens), max_tokens=sum(lens) + case["pad"])
    else:
        st.update(q=rnd(case["B"], H, D, dtype=dt), block_table=table, lengths=torch.tensor(lens, dtype=torch.int32, device=dev))
    return st


# ---------------------------------------------------------------------------------------------------------------
# the operators through the framework, and in their plain form
# ---------------------------------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        return {"packed": _own_packed, "append": _own_append, "gather": _own_gather, "attend": _own_attend}[op](st)
    with torch.no_grad():
        return {"packed": _plain_packed, "append": _plain_append, "gather": _plain_gather, "attend": _plain_attend}[op](st)


def _own_packed(st):
    out = _ft().forgetting_attention_packed(st["q"], st["k"], st["v"], st["log_fgate"], st["cu_seqlens"], st["cu_seqlens_k"])
    return [out.detach(), *torch.autograd.grad([out], st["leaves"], [st["dout"]])] if st["case"]["grad"] else [out]


def _own_append(st):
    _ft().paged_append_8bit(st["k"], st["v"], st["log_fgate"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"], st["log_fgate_pages"], st["slots"])
    return [st[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales", "log_fgate_pages")]


def _own_gather(st):
    return list(_ft().paged_gather(st["k_pages"], st["v_pages"], st["log_fgate_pages"], st["block_table"], st["cu_seqlens"], max_tokens=st["max_tokens"],
                                   k_scales=st["k_scales"], v_scales=st["v_scales"], dtype=_DTYPES[st["case"]["dtype"]]))


def _own_attend(st):
    return [_ft().paged_forgetting_attention_8bit(st["q"], st["k_pages"], st["v_pages"], st["k_scales"], st["v_scales"], st["log_fgate_pages"], st["block_table"],
                                                  st["lengths"])]


def _rows(ends, longest, at_the_end):
    """Places of the tokens of every sequence, (B, longest), the last ones of a row or the first ones, and which of them are tokens."""
    ends = ends.long()
    n = (ends[1:] - ends[:-1])[:, None]
    i = torch.arange(longest, device=ends.device)[None]
    i = i - (longest - n) if at_the_end else i
    real = (i >= 0) & (i < n)
    return torch.where(real, ends[:-1, None] + i, 0), real


def _plain_packed(st):
    c = st["case"]
    H, Hk, D, M, N = c["H"], c["Hk"], c["D"], c["longest"], c["longest"] + c["prefix"]
    B, G, scale = c["B"], H // Hk, D ** -0.5
    ends_k = st["cu_seqlens"] if st["cu_seqlens_k"] is None else st["cu_seqlens_k"]
    at_q, real_q = _rows(st["cu_seqlens"], M, True)            # the last tokens of all sequences stand below each other
    at_k, real_k = _rows(ends_k, N, True)

    def heads(x, at, groups):                                  # (B, Hk, groups * length, D)
        return x[at].float().unflatten(2, (Hk, groups)).permute(0, 2, 3, 1, 4).reshape(B, Hk, groups * at.shape[1], -1)

    def tokens(x, groups, at, real, like):                     # and back, zeros where there is no token
        x = x.reshape(B, Hk, groups, at.shape[1], -1).permute(0, 3, 1, 2, 4).reshape(B, at.shape[1], Hk * groups, -1)
        out = torch.zeros(len(like) + 1, Hk * groups, x.shape[-1], device=x.device)
        out[torch.where(real, at, len(like))] = x
        return out[:-1].reshape(like.shape).to(like.dtype)

    q, k, v = heads(st["q"], at_q, G), heads(st["k"], at_k, 1), heads(st["v"], at_k, 1)
    gates = torch.where(real_k[..., None], st["log_fgate"][at_k], 0.0).double()
    decay = gates.cumsum(1).permute(0, 2, 1).reshape(B, Hk, G, N)
    see = real_k[:, None, :] & real_q[:, :, None] & (torch.arange(N, device=q.device)[None] <= torch.arange(M, device=q.device)[:, None] + (N - M))
    s = torch.matmul(q, k.transpose(-1, -2)).reshape(B, Hk, G, M, N)
    s.mul_(scale)
    ref = decay[..., N - M:N - M + 1]                          # differences from here are small next to the sums themselves
    s += (decay[..., N - M:] - ref).float()[..., None]
    s -= (decay - ref).float()[..., None, :]
    s.masked_fill_(~see[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    p = s.div_(torch.where(total == 0, 1.0, total))
    o = torch.matmul(p.reshape(B, Hk, G * M, N), v)
    out = [tokens(o, G, at_q, real_q, st["q"])]
    if c["grad"]:
        do = heads(st["dout"], at_q, G)
        dv = torch.matmul(p.reshape(B, Hk, G * M, N).transpose(-1, -2), do)
        dp = torch.matmul(do, v.transpose(-1, -2)).reshape(p.shape)
        delta = (do * o).sum(-1).reshape(B, Hk, G, M, 1)
        ds = dp.sub_(delta).mul_(p)
        flat = ds.reshape(B, Hk, G * M, N)
        dq = torch.matmul(flat, k) * scale
        dk = torch.matmul(flat.transpose(-1, -2), q) * scale
        dc = -ds.sum(-2, dtype=torch.float64)
        dc[..., N - M:] += ds.sum(-1, dtype=torch.float64)
        dg = dc.flip(-1).cumsum(-1).flip(-1).float()           # a gate counts for every sum from its own on
        out += [tokens(dq, G, at_q, real_q, st["q"]), tokens(dk, 1, at_k, real_k, st["k"]), tokens(dv, 1, at_k, real_k, st["v"]),
                tokens(dg, G, at_k, real_k, st["log_fgate"])]
    return out


def _plain_append(st):
    c = st["case"]
    S, Hk, D, codes = c["page"], c["Hk"], c["D"], c["codes"]
    G, dev = _block(S), st["slots"].device
    keep = st["slots"] >= 0
    P = st["k_pages"].shape[0]
    blocks = P * S // G
    slot = torch.where(keep, st["slots"], P * S)                          # a spare block takes what has no slot
    block, row = slot // G, slot % G
    # the first row that the step writes in every block: those in front of it stay, in the codes of the new scale
    front = torch.full((blocks + 1,), G, device=dev).scatter_reduce(0, block, row, "amin")[:-1, None, None]
    written = front < G
    for n in ("k", "v"):
        x = st[n].float()
        size = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
        amax = torch.zeros(blocks + 1, Hk, device=dev).scatter_reduce(0, block[:, None].expand(-1, Hk), size, "amax")
        fresh = _scale_of(amax, codes)                                    # (blocks + 1, Hk)
        old = st[n + "_scales"].transpose(1, 2).reshape(blocks, Hk)       # blocks of a page one after the other
        scale = torch.where(written[..., 0], torch.where(front[..., 0] == 0, fresh[:-1], torch.maximum(old, fresh[:-1])), old)
        held = st[n + "_pages"].view(P, Hk, S // G, G, D).transpose(1, 2).reshape(blocks, Hk, G, D).float()
        again = (torch.arange(G, device=dev)[:, None] < front[..., None]) & written[..., None] & (scale != old)[..., None, None]
        held = torch.where(again, held * (old / scale)[..., None, None], held)
        rows = torch.cat([held, held.new_zeros(1, Hk, G, D)])
        rows[block, :, row] = x * (1.0 / torch.cat([scale, scale[:1]]))[block][..., None]
        new = _coded(rows[:-1], codes).view(P, S // G, Hk, G, D).transpose(1, 2).reshape(P, Hk, S, D)
        st[n + "_pages"].copy_(new)
        st[n + "_scales"].copy_(scale.view(P, S // G, Hk).transpose(1, 2))
    flat = torch.cat([st["log_fgate_pages"].transpose(1, 2).reshape(P * S, -1), st["log_fgate"][:1]])
    flat[slot] = st["log_fgate"]
    st["log_fgate_pages"].copy_(flat[:-1].view(P, S, -1).transpose(1, 2))
    return [st[n] for n in ("k_pages", "v_pages", "k_scales", "v_scales", "log_fgate_pages")]


def _values(pages, scales, S):
    """Pages (.., S, D) of codes as the values that they stand for, in 32 bits."""
    G = _block(S)
    return (pages.float().unflatten(-2, (S // G, G)) * scales[..., None, None]).flatten(-3, -2)


def _plain_gather(st):
    c = st["case"]
    S, dt, ends = c["page"], _DTYPES[c["dtype"]], st["cu_seqlens"].long()
    t = torch.arange(st["max_tokens"], device=ends.device)
    b = (torch.searchsorted(ends, t, right=True) - 1).clamp(max=c["B"] - 1)
    real = (t < ends[-1])[:, None]
    pos = torch.where(real[:, 0], t - ends[b], 0)
    page, row = st["block_table"][b, pos // S].long(), pos % S
    G = _block(S)
    out = []
    for n in ("k", "v"):
        x = st[n + "_pages"][page, :, row].float() * st[n + "_scales"][page, :, row // G][..., None]
        out.append(torch.where(real[..., None], x, 0.0).to(dt))
    return out + [torch.where(real, st["log_fgate_pages"][page, :, row], 0.0)]


def _plain_attend(st):
    c = st["case"]
    B, H, Hk, D, S = (c[n] for n in ("B", "H", "Hk", "D", "page"))
    table, lengths = st["block_table"].long(), st["lengths"].long()
    N = table.shape[1] * S
    valid = (torch.arange(N, device=table.device) < lengths[:, None])[:, None]                    # (B, 1, N)
    gates = st["log_fgate_pages"][table].transpose(1, 2).reshape(B, H, N).double() * valid
    behind = (gates.flip(-1).cumsum(-1).flip(-1) - gates).float()                                 # of the keys behind each key
    k = _values(st["k_pages"][table], st["k_scales"][table], S).transpose(1, 2).reshape(B, Hk, N, D)
    s = torch.matmul(st["q"].float().view(B, Hk, H // Hk, D), k.transpose(-1, -2)).view(B, H, N) / math.sqrt(D) + behind
    del k
    s = s.masked_fill(~valid, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = (s - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    v = _values(st["v_pages"][table], st["v_scales"][table], S).transpose(1, 2).reshape(B, Hk, N, D)
    return [torch.matmul(p.view(B, Hk, H // Hk, N), v).view(B, H, D).to(st["q"].dtype)]


# ---------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"packed": _exact_packed, "append": _exact_append, "gather": _exact_gather, "attend": _exact_attend}[case["op"]](st)


def _exact_packed(st):
    """Sequence by sequence and head by head, gradients by 64-bit automatic differentiation."""
    c = st["case"]
    new, front = _sequences(c)
    H, group = c["H"], c["H"] // c["Hk"]
    names = ("q", "k", "v", "log_fgate")
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    grads = [torch.zeros_like(st[n], dtype=torch.float64) for n in names]
    q0 = k0 = 0
    for m, f in zip(new, front):
        n = m + f
        for h in range(H if m else 0):
            cut = [st["q"][q0:q0 + m, h], st["k"][k0:k0 + n, h // group], st["v"][k0:k0 + n, h // group], st["log_fgate"][k0:k0 + n, h]]
            q, k, v, g = (x.detach().double().requires_grad_() for x in cut)
            decay = g.cumsum(0)
            s = q @ k.t() / math.sqrt(c["D"]) + (decay[n - m:, None] - decay[None])
            s = s.masked_fill(torch.ones(m, n, dtype=torch.bool, device=s.device).triu(n - m + 1), -math.inf)
            with torch.set_grad_enabled(c["grad"]):
                o = torch.softmax(s, -1) @ v
            out[q0:q0 + m, h] = o.detach()
            if c["grad"]:
                dq, dk, dv, dg = torch.autograd.grad(o, (q, k, v, g), st["dout"][q0:q0 + m, h].double())
                grads[0][q0:q0 + m, h] = dq
                grads[1][k0:k0 + n, h // group] += dk
                grads[2][k0:k0 + n, h // group] += dv
                grads[3][k0:k0 + n, h] = dg
        q0, k0 = q0 + m, k0 + n
    return [out] + grads if c["grad"] else [out]


def _nearest(x, codes):
    """64-bit values to the nearest code, ties to the even one: e4m3 has steps of an eighth of the power of two below, at least 2^-9."""
    if codes == "int8":
        return x.round()
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))) / 8
    return (x / step).round() * step


def _exact_append(st):
    """Run by run: the tokens of a block one after the other in the step."""
    c = st["case"]
    S, codes = c["page"], c["codes"]
    G = _block(S)
    slots = st["slots"].tolist()
    runs = []
    for t, s in enumerate(slots):
        if s < 0:
            continue
        if runs and runs[-1][-1] == t - 1 and slots[t - 1] == s - 1 and s % G:
            runs[-1].append(t)
        else:
            runs.append([t])
    if len(runs) > 4000:
        return None
    out = {}
    for n in ("k", "v"):
        pages, scales = st[n + "_pages"].double(), st[n + "_scales"].double()
        for r in runs:
            x = st[n][r[0]:r[-1] + 1].double().transpose(0, 1)              # (Hk, tokens, D)
            page, row = slots[r[0]] // S, slots[r[0]] % S
            b, first = row // G, row - row % G
            need = (x.abs().amax((1, 2)) / _LARGEST[codes]).clamp(min=2.0 ** -126)
            scale = torch.exp2(torch.ceil(torch.log2(need)))
            if row % G:
                scale = torch.maximum(scale, scales[page, :, b])
                held = pages[page, :, first:row]
                pages[page, :, first:row] = _nearest(held * (scales[page, :, b] / scale)[:, None, None], codes)
            pages[page, :, row:row + len(r)] = _nearest(x / scale[:, None, None], codes)
            scales[page, :, b] = scale
        out[n] = pages, scales
    gates = st["log_fgate_pages"].double()
    has = st["slots"] >= 0
    at = st["slots"][has]
    gates[at // S, :, at % S] = st["log_fgate"][has].double()
    return [out["k"][0], out["v"][0], out["k"][1], out["v"][1], gates]


def _request_rows(st, b, n, names, block):
    """The first n cached tokens of request b, (heads, n, ..), in 64 bits."""
    S = st["case"]["page"]
    ids = st["block_table"][b, :(n + S - 1) // S].long()
    rows = []
    for name in names:
        x = st[name][ids].double()
        if name != "log_fgate_pages":
            x = x * st[name[0] + "_scales"][ids].double().repeat_interleave(block, -1)[..., None]
        rows.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
    return rows


def _exact_gather(st):
    c = st["case"]
    T = st["max_tokens"]
    names = ("k_pages", "v_pages", "log_fgate_pages")
    out = [torch.zeros(T, st[n].shape[1], *st[n].shape[3:], dtype=torch.float64, device=st[n].device) for n in names]
    at = 0
    for b, n in enumerate(_lengths(c)):
        for o, x in zip(out, _request_rows(st, b, n, names, _block(c["page"]))):
            o[at:at + n] = x.transpose(0, 1)
        at += n
    return out


def _exact_attend(st):
    """Request by request over the keys that it holds."""
    c = st["case"]
    group = c["H"] // c["Hk"]
    out = torch.zeros_like(st["q"], dtype=torch.float64)
    for b, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        k, v, g = _request_rows(st, b, n, ("k_pages", "v_pages", "log_fgate_pages"), _block(c["page"]))
        decay = g.cumsum(-1)
        q = st["q"][b].double().view(c["Hk"], group, -1)
        s = torch.matmul(q, k.transpose(-1, -2)).flatten(0, 1) * c["D"] ** -0.5 + (decay[:, -1:] - decay)
        out[b] = torch.matmul(torch.softmax(s, -1).view(c["Hk"], group, n), v).flatten(0, 1)
    return [out]


def work(case):
    op, H, Hk, D = case["op"], case["H"], case["Hk"], case["D"]
    if op == "packed":
        new, front = _sequences(case)
        T, N = sum(new), sum(new) + sum(front)
        pairs = H * sum(m * f + m * (m + 1) // 2 for m, f in zip(new, front))    # queries with the keys that they see
        rows, keys, gate = 2 * T * H * D, 2 * N * Hk * D, 4 * N * H
        if case["grad"]:
            return {"bytes": 4 * rows + 4 * keys + 2 * gate, "flops": 14 * pairs * D}
        return {"bytes": 2 * rows + 2 * keys + gate, "flops": 4 * pairs * D}
    if op == "append":
        T = case["T"] - case["skipped"]
        return {"bytes": 6 * T * Hk * D + 8 * T * H + 8 * case["T"] + 8 * T * Hk // 16, "flops": 4 * T * Hk * D}
    keys = sum(_lengths(case))
    scales, table = 8 * keys * Hk // _block(case["page"]), 4 * keys // case["page"]
    if op == "gather":
        return {"bytes": 6 * keys * Hk * D + 8 * keys * H + scales + table, "flops": 2 * keys * Hk * D}
    return {"bytes": 2 * keys * Hk * D + 4 * keys * H + scales + table + 4 * case["B"] * H * D, "flops": 4 * keys * H * D}
