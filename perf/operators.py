"""Cases of the cache operators: key/query norm with rotation, page forking and
compaction, and decode attention over a shared INT4 prefix.

``run`` computes an operator in plain torch (``own`` false) or calls the
library (``own`` true) on the state that ``prepare`` makes; ``exact`` gives the
floating results in 64 bits. The INT4 pages are built here from the layout that
include/hetero_kv.h documents, so nothing of the library is needed for them.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda"
D = 128
BLOCK = 128  # tokens of a page block
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ------------------------------------------------------------------ page layout
def _nibble_tables():
    """For the 16,384 nibbles of a block's K (and V) codes, low nibble of a byte
    first: which element (token * 128 + dim) each one holds."""
    n = np.arange(2 * 8192)
    byte, half = n // 2, n % 2
    t, y = byte // 64, byte % 64
    j, w, k = y // 16, (y // 4) % 4, 2 * (y % 4) + half
    k_of = t * D + 16 * (2 * w + (k % 4) // 2) + 8 * (k % 2) + 2 * j + k // 4
    pair, pos = byte // 128, (byte % 128) // 16
    y = ((pos - 2 * pair) % 8) * 16 + byte % 16
    i, e4, k = y // 16, (y // 4) % 4, 2 * (y % 4) + half
    e = 4 * e4 + k % 4
    v_of = (2 * pair + k // 4) * D + 16 * (e // 2) + 8 * (e % 2) + i
    return k_of, v_of


_K_OF, _V_OF = _nibble_tables()
_K_AT, _V_AT = np.argsort(_K_OF), np.argsort(_V_OF)


def _table(a):
    return torch.from_numpy(a).to(DEV)


def block_bytes(fmt, group):
    ng = D // group
    return BLOCK * (128 + 8 * ng + (2 * ng if fmt == "ref" else 0))


def _quantise(x, fmt, group):
    """Codes [N, 128, 128] and the two metadata arrays [N, 128, ng] of x [N, 128, 128]."""
    g = x.float().view(x.shape[0], BLOCK, D // group, group)
    lo, hi = g.amin(-1), g.amax(-1)
    if fmt == "ref":
        a = ((hi - lo) / 15).clamp_min(1e-8)
        b = (-lo / a).round().clamp(0, 15)
        c = (g / a[..., None] + b[..., None]).round()
        b = b.to(torch.uint8)
    else:
        a, b = ((hi - lo) / 15).half(), lo.half()
        c = ((g - b.float()[..., None]) / a.float()[..., None]).round()
    return c.clamp(0, 15).to(torch.uint8).view(x.shape), a, b


def _pack(k, v, fmt, group):
    """Page blocks [N, block_bytes] of K and V [N, 128, 128]."""
    n, ng = k.shape[0], D // group
    parts = []
    ck, ka, kb = _quantise(k, fmt, group)
    cv, va, vb = _quantise(v, fmt, group)
    for c, at in ((ck, _K_OF), (cv, _V_OF)):
        nib = c.view(n, -1).index_select(1, _table(at)).view(n, 8192, 2)
        parts.append(nib[..., 0] | (nib[..., 1] << 4))
    if fmt == "ref":
        metas = [ka, va, kb, vb]
    else:  # V: the two tokens of a pair side by side
        pair = [m.view(n, 64, 2, ng).transpose(2, 3) for m in (va, vb)]
        metas = [ka, kb] + pair
    parts += [m.reshape(n, -1).contiguous().view(torch.uint8).view(n, -1) for m in metas]
    return torch.cat(parts, 1)


def _unpack(blocks, fmt, group):
    """K and V [N, 128, 128] in 32 bits of page blocks [N, block_bytes]."""
    n, ng = blocks.shape[0], D // group
    out = []
    meta = blocks[:, 16384:].contiguous()
    for role, at in ((0, _K_AT), (1, _V_AT)):
        raw = blocks[:, 8192 * role:8192 * (role + 1)]
        nib = torch.stack((raw & 15, raw >> 4), -1).view(n, 16384)
        c = nib.index_select(1, _table(at)).float().view(n, BLOCK, ng, group)
        if fmt == "ref":
            s = meta[:, :1024 * ng].contiguous().view(torch.float32).view(n, 2, BLOCK, ng, 1)[:, role]
            z = meta[:, 1024 * ng:].reshape(n, 2, BLOCK, ng, 1)[:, role].float()
            x = (c - z) * s
        else:
            h = meta.view(torch.float16).view(n, 2, 2, -1)[:, role].float()  # scales | mins
            h = (h.view(n, 2, BLOCK, ng, 1) if role == 0
                 else h.view(n, 2, 64, ng, 2).transpose(3, 4).reshape(n, 2, BLOCK, ng, 1))
            x = c * h[:, 0] + h[:, 1]
        out.append(x.view(n, BLOCK, D))
    return out


def _fill_pages(gen, pages, per_page, fmt, group):
    """A pool [pages, page_bytes] of quantised keys and values as a model has
    them: about N(0, 1), with a few key channels ten times as large."""
    chunks = []
    for lo in range(0, pages * per_page, 4096):
        n = min(4096, pages * per_page - lo)
        k = torch.randn(n, BLOCK, D, generator=gen, device=DEV)
        v = torch.randn(n, BLOCK, D, generator=gen, device=DEV)
        k[..., 5::37] *= 10
        chunks.append(_pack(k, v, fmt, group))
    return torch.cat(chunks).view(pages, -1)


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _ints(text):
    return [int(x) for x in str(text).split(",")]


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 8 sequences, 32 query and 8 KV heads: launch latency
        dict(name="norm_rope step", op="norm_rope", B=8, T=1, Hq=32, Hkv=8, rot=128, adjacent=False, norm=True, dtype="bf16"),
        # a small ragged batch, half of each head rotated, pairs of neighbours, no norm
        dict(name="norm_rope partial", op="norm_rope", B=3, T=777, Hq=28, Hkv=4, rot=64, adjacent=True, norm=False, dtype="f16"),
        # one chunk of a chunked prefill (28 query, 4 KV heads)
        dict(name="norm_rope chunk", op="norm_rope", B=1, T=4096, Hq=28, Hkv=4, rot=128, adjacent=False, norm=True, dtype="bf16"),
        # a whole 32K prompt at once
        dict(name="norm_rope prompt", op="norm_rope", B=1, T=32768, Hq=32, Hkv=8, rot=128, adjacent=False, norm=True, dtype="f16"),
        # four samples of one short prompt: a page per head and new sample
        dict(name="fork 4", op="fork", B=4, H=8, roots=1, tokens=1000, page_tokens=256, fmt="fp16min", group=32),
        # eight long prompts forked to 64 sequences
        dict(name="fork 64", op="fork", B=64, H=8, roots=8, tokens=31685, page_tokens=256, fmt="fp16min", group=32),
        # a few short sequences moved out of a scattered pool
        dict(name="compact 3", op="compact", B=3, H=4, roots=2, tokens=2900, page_tokens=128, fmt="ref", group=128),
        # 16 sequences of 31,680 tokens: a pool of 0.65 GB put in order
        dict(name="compact 16", op="compact", B=16, H=8, roots=16, tokens=31680, page_tokens=256, fmt="fp16min", group=32),
        # a few samples of a short prompt: launch latency
        dict(name="shared 4", op="shared", groups="4", Hkv=4, G=7, prefix="1000", body=100, dense=96, page_tokens=128, fmt="ref", group=32, dtype="f16"),
        # 8 samples of one 32K prompt, 1,088 dense tokens each
        dict(name="shared 8", op="shared", groups="8", Hkv=8, G=4, prefix="31680", body=512, dense=1088, page_tokens=256, fmt="fp16min", group=32, dtype="bf16"),
        # prompts of several lengths with samples of each, one alone
        dict(name="shared ragged", op="shared", groups="11,1,7", Hkv=8, G=5, prefix="9001,300,16385", body=333, dense=577, page_tokens=128, fmt="ref", group=64, dtype="f16"),
        # a batch of 64 over one system prompt of 128K tokens
        dict(name="shared 64", op="shared", groups="64", Hkv=8, G=4, prefix="131072", body=256, dense=1088, page_tokens=256, fmt="fp16min", group=32, dtype="bf16"),
    ]


def _between(rng, lo, hi):
    """A whole number of [lo, hi], its logarithm spread evenly."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm_rope", "fork", "compact", "shared"])
    fmt, group = rng.choice(["ref", "fp16min"]), rng.choice([32, 64, 128])
    page_tokens = rng.choice([128, 256])
    if op == "norm_rope":
        Hkv = rng.choice([1, 2, 4, 8])
        Hq = Hkv * rng.randint(1, 8)
        rows = _between(rng, 1, 32768 * 40 // (Hq + Hkv))
        B = rng.randint(1, min(16, rows))
        return dict(op=op, B=B, T=max(1, min(rows, 32768) // B), Hq=Hq, Hkv=Hkv, rot=2 * rng.randint(1, 64), adjacent=rng.random() < 0.5,
                    norm=rng.random() < 0.7, dtype=rng.choice(["bf16", "f16"]))
    if op in ("fork", "compact"):
        H, B = rng.choice([1, 2, 4, 8]), rng.randint(2, 64 if op == "fork" else 16)
        return dict(op=op, B=B, H=H, roots=rng.randint(1, B), tokens=_between(rng, 1, 31680), page_tokens=page_tokens, fmt=fmt, group=group)
    P, G = rng.randint(1, 4), rng.randint(1, 8)
    groups = [_between(rng, 1, 16) for _ in range(P)]
    return dict(op=op, groups=",".join(map(str, groups)), Hkv=rng.choice([1, 2, 4, 8]), G=G,
                prefix=",".join(str(_between(rng, 1, 32768)) for _ in range(P)), body=rng.choice([0, _between(rng, 1, 1000)]),
                dense=_between(rng, 1, 1088), page_tokens=page_tokens, fmt=fmt, group=group, dtype=rng.choice(["bf16", "f16"]))


# ------------------------------------------------------------------ states
def prepare(case, seed):
    return {"norm_rope": _prepare_norm_rope, "fork": _prepare_pages, "compact": _prepare_pages, "shared": _prepare_shared}[case["op"]](case, _gen(seed))


def _prepare_norm_rope(c, gen):
    B, T, Hq, Hkv, dt = c["B"], c["T"], c["Hq"], c["Hkv"], TYPES[c["dtype"]]
    # the packed projection of a layer: queries, keys and values of a token side by side
    qkv = (torch.randn(B, T, (Hq + 2 * Hkv) * D, generator=gen, device=DEV) * 2).to(dt).view(B, T, Hq + 2 * Hkv, D)
    start = torch.randint(0, 1024, (B, 1), generator=gen, device=DEV)
    ang = torch.outer(torch.arange(T + 1024, device=DEV, dtype=torch.float64),
                      torch.tensor(1e6, device=DEV, dtype=torch.float64) ** (-torch.arange(0, c["rot"], 2, device=DEV, dtype=torch.float64) / c["rot"]))
    w = [(1 + 0.2 * torch.randn(D, generator=gen, device=DEV)).to(dt) if c["norm"] else None for _ in range(2)]
    return dict(op="norm_rope", q=qkv[:, :, :Hq].transpose(1, 2), k=qkv[:, :, Hq:Hq + Hkv].transpose(1, 2),
                pos=(start + torch.arange(T, device=DEV)).to(torch.int32), table=torch.cat((ang.cos(), ang.sin()), 1).float(),
                qw=w[0], kw=w[1], adjacent=c["adjacent"])


def _roots(c):
    """Root sequence of each of the B sequences: the first `roots` are their own."""
    B, R = c["B"], c["roots"]
    return [b if b < R else (b - R) % R for b in range(B)]


def _prepare_pages(c, gen):
    B, H, P = c["B"], c["H"], c["page_tokens"]
    roots = _roots(c)
    lens = [max(1, c["tokens"] - 97 * r) for r in range(c["roots"])]
    maxp = -(-c["tokens"] // P) + 2
    live = sum(-(-n // P) for n in lens) * H
    pages = live + B * H + live // 8 + 8
    pool = torch.randint(0, 256, (pages, P // BLOCK * block_bytes(c["fmt"], c["group"])), dtype=torch.uint8, generator=gen, device=DEV)
    ids = torch.randperm(pages, generator=gen, device=DEV).to(torch.int32)
    table = torch.full((B, H, maxp), -1, dtype=torch.int32, device=DEV)
    at = 0
    for r, n in enumerate(lens):
        k = -(-n // P)
        table[r, :, :k] = ids[at:at + H * k].view(H, k)
        at += H * k
    lengths = torch.zeros(B, dtype=torch.int32, device=DEV)
    lengths[:c["roots"]] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s = dict(op=c["op"], pool=pool, table=table.view(B * H, maxp), lengths=lengths, parents=torch.tensor(roots, dtype=torch.int32, device=DEV),
             H=H, P=P, fmt=c["fmt"], group=c["group"], bb=block_bytes(c["fmt"], c["group"]), max_len=max(lens))
    if c["op"] == "compact":
        # sequences forked from the same root share its full pages, as forking leaves them
        more = ids[at:]
        t3, n = s["table"].view(B, H, maxp), 0
        for b in range(c["roots"], B):
            r = roots[b]
            t3[b], lengths[b] = t3[r], lengths[r]
            if lens[r] % P:
                t3[b, :, lens[r] // P] = more[n:n + H]
                n += H
    used = s["table"][s["table"] >= 0].long()
    s["refs"] = torch.zeros(pages, dtype=torch.int32, device=DEV).index_add_(0, used, torch.ones_like(used, dtype=torch.int32))
    if c["op"] == "compact":
        s["into"] = dict(pool=torch.zeros_like(pool), table=torch.full_like(s["table"], -1), lengths=torch.zeros_like(lengths), refs=torch.zeros_like(s["refs"]))
    return s


def _paged(gen, units, most, P, fmt, group):
    """A pool with room for `most` tokens of each unit and its shuffled page table."""
    per = max(1, -(-most // P))
    table = torch.randperm(units * per, generator=gen, device=DEV).to(torch.int32).view(units, per)
    return _fill_pages(gen, units * per, P // BLOCK, fmt, group), table


def _prepare_shared(c, gen):
    groups, prefix, H, P, dt = _ints(c["groups"]), _ints(c["prefix"]), c["Hkv"], c["page_tokens"], TYPES[c["dtype"]]
    B = sum(groups)
    s = dict(op="shared", starts=[sum(groups[:i]) for i in range(len(groups) + 1)], prefix_most=max(prefix), body_most=c["body"], dense_most=c["dense"],
             H=H, P=P, fmt=c["fmt"], group=c["group"], dtype=dt)
    s["q"] = torch.randn(B, H * c["G"], D, generator=gen, device=DEV).to(dt)
    s["prefix_pool"], s["prefix_table"] = _paged(gen, len(prefix) * H, max(prefix), P, c["fmt"], c["group"])
    s["prefix_lengths"] = torch.tensor(prefix, dtype=torch.int32, device=DEV)
    # the samples of a prompt have got to different lengths
    drop = torch.rand(B, generator=gen, device=DEV) * 0.25
    if c["body"]:
        s["body_pool"], s["body_table"] = _paged(gen, B * H, c["body"], P, c["fmt"], c["group"])
        s["body_lengths"] = (c["body"] * (1 - drop)).to(torch.int32)
    s["dense_k"], s["dense_v"] = (torch.randn(B, H, c["dense"], D, generator=gen, device=DEV).to(dt) for _ in range(2))
    s["dense_lengths"] = torch.full((B,), c["dense"], dtype=torch.int32, device=DEV)
    return s


# ------------------------------------------------------------------ plain forms
def _norm_rope_plain(s):
    cs = s["table"][s["pos"].long()][:, None]  # [B, 1, T, rot]
    r = cs.shape[-1] // 2
    cos, sin = cs[..., :r], cs[..., r:]

    def one(x, w):
        y = x.float()
        if w is not None:
            y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        a, b = (y[..., 0:2 * r:2], y[..., 1:2 * r:2]) if s["adjacent"] else (y[..., :r], y[..., r:2 * r])
        p, m = a * cos - b * sin, b * cos + a * sin
        rot = torch.stack((p, m), -1).flatten(-2) if s["adjacent"] else torch.cat((p, m), -1)
        return torch.cat((rot, y[..., 2 * r:]), -1).to(x.dtype)

    return one(s["q"], s["qw"]), one(s["k"], s["kw"])


def _fork_plain(s):
    table, lengths, refs, pool, P, H = s["table"], s["lengths"], s["refs"], s["pool"], s["P"], s["H"]
    B, maxp = lengths.numel(), table.shape[1]
    par = s["parents"].long()
    b = torch.arange(B, device=DEV)
    first = torch.full((B,), B, device=DEV).scatter_reduce_(0, par, b, "amin")
    keeps = (first[par] == b)[:, None, None]
    old = table.view(B, H, maxp)
    n = lengths[par]
    i = torch.arange(maxp, device=DEV)
    full = i < (n // P)[:, None, None]
    new = torch.where(keeps | full, old[par], -1)
    refs.index_add_(0, old.reshape(-1).clamp_min(0).long(), -(old.reshape(-1) >= 0).int())
    refs.index_add_(0, new.reshape(-1).clamp_min(0).long(), (new.reshape(-1) >= 0).int())
    # a partly filled last page that another sequence keeps is copied to the lowest free page
    part = (n % P > 0)[:, None] & ~keeps[..., 0].expand(B, H)
    at = (n // P).long()[:, None, None].expand(B, H, 1)
    src = old[par].gather(2, at.clamp_max(maxp - 1))[..., 0]
    free = torch.argsort((refs != 0).to(torch.uint8), stable=True)
    rank = part.reshape(-1).long().cumsum(0) - 1
    dst = torch.where(part, free[rank.clamp_min(0)].view(B, H).int(), src)
    new.scatter_(2, at.clamp_max(maxp - 1), torch.where(part, dst, new.gather(2, at.clamp_max(maxp - 1))[..., 0])[..., None])
    refs.index_add_(0, dst.reshape(-1).clamp_min(0).long(), part.reshape(-1).int())
    blocks = pool.view(-1, s["bb"])
    bp = P // BLOCK
    k = torch.arange(bp, device=DEV)
    used = part[..., None] & (k * BLOCK < (n % P)[:, None, None])
    frm = src[..., None].clamp_min(0).long() * bp + k
    to = torch.where(used, dst[..., None].long() * bp + k, frm)
    blocks.index_copy_(0, to.reshape(-1), blocks[frm.reshape(-1)])
    table.copy_(new.view_as(table))
    lengths.copy_(n)
    return dict(pool=pool, table=table, lengths=lengths, refs=refs)


def _compact_plain(s):
    t, into = s["table"].reshape(-1).long(), s["into"]
    pages, maxp = s["pool"].shape[0], s["table"].shape[1]
    e = torch.arange(t.numel(), device=DEV)
    first = torch.full((pages,), t.numel(), device=DEV).scatter_reduce_(0, t.clamp_min(0), torch.where(t >= 0, e, t.numel()), "amin")
    is_first = (t >= 0) & (first[t.clamp_min(0)] == e)
    rank = is_first.long().cumsum(0) - 1
    new = torch.where(t >= 0, rank[first[t.clamp_min(0)].clamp_max(t.numel() - 1)], -1)
    into["table"].copy_(new.view_as(s["table"]))
    into["refs"].zero_().index_add_(0, new.clamp_min(0), (t >= 0).int())
    into["lengths"].copy_(s["lengths"])
    n = s["lengths"].repeat_interleave(s["H"])[:, None]
    held = (torch.arange(maxp, device=DEV) * s["P"] < n).reshape(-1) & is_first
    into["pool"].index_copy_(0, new[held], s["pool"][t[held]])
    return dict(into)


def _tokens(pool, table, P, fmt, group):
    """K and V [units, capacity, 128] in 32 bits through a page table."""
    u, per = table.shape
    blocks = pool[table.reshape(-1).clamp_min(0).long()].view(u * per * (P // BLOCK), -1)
    return [x.view(u, per * P, D) for x in _unpack(blocks, fmt, group)]


def _shared_plain(s):
    q, H, P = s["q"].float(), s["H"], s["P"]
    B, G, N = q.shape[0], q.shape[1] // H, len(s["starts"]) - 1
    q = q.view(B, H, G, D) / math.sqrt(D)
    start = torch.tensor(s["starts"], device=DEV)
    most = max(y - x for x, y in zip(s["starts"], s["starts"][1:]))
    pid = torch.searchsorted(start[1:], torch.arange(B, device=DEV), right=True)
    slot = torch.arange(B, device=DEV) - start[pid]
    rows = torch.zeros(N, most, H, G, D, device=DEV)
    rows[pid, slot] = q
    rows = rows.transpose(1, 2).reshape(N, H, most * G, D)
    k, v = (x.view(N, H, -1, D) for x in _tokens(s["prefix_pool"], s["prefix_table"], P, s["fmt"], s["group"]))
    x = rows @ k.transpose(-1, -2)
    x.masked_fill_((torch.arange(k.shape[2], device=DEV) >= s["prefix_lengths"][:, None])[:, None, None], -math.inf)
    m1 = x.amax(-1, keepdim=True)
    p = torch.exp(x - m1)
    o1, l1, m1 = (y.view(N, H, most, G, -1).transpose(1, 2)[pid, slot] for y in (p @ v, p.sum(-1, keepdim=True), m1))
    ks, vs, ns = [s["dense_k"].float()], [s["dense_v"].float()], [s["dense_lengths"]]
    if s["body_most"]:
        k, v = (x.view(B, H, -1, D) for x in _tokens(s["body_pool"], s["body_table"], P, s["fmt"], s["group"]))
        ks.append(k), vs.append(v), ns.append(s["body_lengths"])
    hide = torch.cat([torch.arange(k.shape[2], device=DEV) >= n[:, None] for k, n in zip(ks, ns)], 1)
    x = q @ torch.cat(ks, 2).transpose(-1, -2)
    x.masked_fill_(hide[:, None, None], -math.inf)
    m2 = x.amax(-1, keepdim=True)
    p = torch.exp(x - m2)
    o2, l2 = p @ torch.cat(vs, 2), p.sum(-1, keepdim=True)
    m = torch.maximum(m1, m2)
    a, b = torch.exp(m1 - m), torch.exp(m2 - m)
    return ((o1 * a + o2 * b) / (l1 * a + l2 * b)).view(B, H * G, D).to(s["dtype"])


# ------------------------------------------------------------------ the library's calls
def _handle(s):
    """The stores and pools over the state's memory, which a program makes once and keeps."""
    h = s.get("handle")
    if h is None:
        from hetero_kvcache_optimizer_b200 import kvstore as kv
        from hetero_kvcache_optimizer_b200.memory.page_pool import PagePool

        def store(pool, table, lengths, most):
            return kv.Int4KVStore.wrap(pool, table, lengths, s["H"], fmt=s["fmt"], group=s["group"], page_tokens=s["P"], len_hint=most)

        h = s["handle"] = {"kv": kv}
        if s["op"] in ("fork", "compact"):
            h["pages"] = PagePool(store(s["pool"], s["table"], s["lengths"], s["max_len"]), refs=s["refs"])
            if s["op"] == "compact":
                t = s["into"]
                h["into"] = PagePool(store(t["pool"], t["table"], t["lengths"], s["max_len"]), refs=t["refs"])
        elif s["op"] == "shared":
            h["prefix"] = kv.SharedPrefix(store(s["prefix_pool"], s["prefix_table"], s["prefix_lengths"], s["prefix_most"]), s["starts"])
            h["body"] = store(s["body_pool"], s["body_table"], s["body_lengths"], s["body_most"]) if s["body_most"] else None
            h["dense"] = kv.DenseKV(s["q"].shape[0], s["H"], s["dense_most"], dtype=s["dtype"], k=s["dense_k"], v=s["dense_v"])
            h["dense"].set_lengths(s["dense_most"])
    return h


def _run_own(s):
    h = _handle(s)
    if s["op"] == "norm_rope":
        return h["kv"].norm_rope(s["q"], s["k"], s["pos"], s["table"], s["qw"], s["kw"], eps=1e-6, adjacent=s["adjacent"])
    if s["op"] == "fork":
        h["pages"].fork(s["parents"])
        return dict(pool=s["pool"], table=s["table"], lengths=s["lengths"], refs=s["refs"])
    if s["op"] == "compact":
        h["pages"].compact(h["into"])
        return dict(s["into"])
    return h["kv"].decode_shared(s["q"], h["prefix"], h["body"], h["dense"], out_dtype=s["dtype"])


def run(state):
    if own:
        return _run_own(state)
    return {"norm_rope": _norm_rope_plain, "fork": _fork_plain, "compact": _compact_plain, "shared": _shared_plain}[state["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "norm_rope":
        rows = c["B"] * c["T"] * (c["Hq"] + c["Hkv"])
        return {"bytes": rows * D * 4 + c["B"] * c["T"] * (4 + 4 * c["rot"]), "flops": rows * (4 * D + 3 * c["rot"])}
    if c["op"] == "fork":
        lens = [max(1, c["tokens"] - 97 * r) for r in range(c["roots"])]
        P, bb = c["page_tokens"], block_bytes(c["fmt"], c["group"])
        blocks = sum(-(-(lens[r] % P) // BLOCK) for b, r in enumerate(_roots(c)) if b != r) * c["H"]
        entries = c["B"] * c["H"] * (-(-c["tokens"] // P) + 2)
        return {"bytes": 2 * blocks * bb + 8 * entries, "flops": 0}
    if c["op"] == "compact":
        lens = [max(1, c["tokens"] - 97 * r) for r in range(c["roots"])]
        P, bb = c["page_tokens"], block_bytes(c["fmt"], c["group"])
        pages = sum(-(-n // P) for n in lens) + sum(lens[r] % P > 0 for b, r in enumerate(_roots(c)) if b != r)
        entries = c["B"] * c["H"] * (-(-c["tokens"] // P) + 2)
        return {"bytes": 2 * pages * c["H"] * (P // BLOCK) * bb + 8 * entries, "flops": 0}
    groups, prefix, H, G = _ints(c["groups"]), _ints(c["prefix"]), c["Hkv"], c["G"]
    B, tok = sum(groups), block_bytes(c["fmt"], c["group"]) / BLOCK
    seen = sum(n * t for n, t in zip(groups, prefix)) + B * (c["body"] * 0.875 + c["dense"])
    return {"bytes": H * tok * (sum(prefix) + B * c["body"] * 0.875) + B * H * c["dense"] * 4 * D + B * H * G * D * 4, "flops": 4 * D * H * G * seen}


# ------------------------------------------------------------------ in 64 bits
def exact(case, seed):
    if case["op"] in ("fork", "compact"):
        return None  # whole numbers alone
    s = prepare(case, seed)
    return _exact_norm_rope(s) if case["op"] == "norm_rope" else _exact_shared(s)


def _exact_norm_rope(s):
    """Each pair of coordinates as a complex number, turned by cos + i sin."""
    r = s["table"].shape[1] // 2
    turn = torch.complex(s["table"][:, :r].double(), s["table"][:, r:].double())[s["pos"].long()]
    out = []
    for x, w in ((s["q"], s["qw"]), (s["k"], s["kw"])):
        y = torch.empty(x.shape, dtype=torch.float64, device=DEV)
        for h in range(x.shape[1]):
            z = x[:, h].double()
            if w is not None:
                z = z / torch.sqrt((z * z).sum(-1, keepdim=True) / D + 1e-6) * w.double()
            first = slice(0, 2 * r, 2) if s["adjacent"] else slice(0, r)
            second = slice(1, 2 * r, 2) if s["adjacent"] else slice(r, 2 * r)
            c = torch.complex(z[..., first], z[..., second]) * turn
            z[..., first], z[..., second] = c.real, c.imag
            y[:, h] = z
        out.append(y)
    return tuple(out)


def _exact_unit(pool, pages, n, s):
    """K and V [n, 128] in 64 bits of one unit's first n tokens: each nibble put at its place."""
    P, ng, group = s["P"], D // s["group"], s["group"]
    used = pages[:-(-n // P)].long()
    raw = pool[used].view(-1, block_bytes(s["fmt"], group))
    N = raw.shape[0]
    res = []
    for role, of in ((0, _K_OF), (1, _V_OF)):
        code = raw[:, 8192 * role:8192 * role + 8192].to(torch.int32)
        x = torch.empty(N, BLOCK * D, dtype=torch.float64, device=DEV)
        x[:, _table(of[0::2])] = (code % 16).double()
        x[:, _table(of[1::2])] = (code // 16).double()
        x = x.view(N, BLOCK, ng, group)
        if s["fmt"] == "ref":
            a = raw[:, 16384 + 512 * ng * role:][:, :512 * ng].contiguous().view(torch.float32).double().view(N, BLOCK, ng, 1)
            b = raw[:, 16384 + 1024 * ng + 128 * ng * role:][:, :128 * ng].double().reshape(N, BLOCK, ng, 1)
            x = a * (x - b)
        else:
            a, b = (raw[:, 16384 + 512 * ng * role + 256 * ng * j:][:, :256 * ng].contiguous().view(torch.float16).double() for j in (0, 1))
            if role:
                a, b = (y.view(N, 64, ng, 2).permute(0, 1, 3, 2) for y in (a, b))
            x = a.reshape(N, BLOCK, ng, 1) * x + b.reshape(N, BLOCK, ng, 1)
        res.append(x.reshape(-1, D)[:n])
    return res


def _exact_shared(s):
    q, H = s["q"].double(), s["H"]
    B, G = q.shape[0], q.shape[1] // H
    n_prefix, n_dense = s["prefix_lengths"].tolist(), s["dense_lengths"].tolist()
    n_body = s["body_lengths"].tolist() if s["body_most"] else [0] * B
    out = torch.empty(B, H, G, D, dtype=torch.float64, device=DEV)
    for g in range(len(n_prefix)):
        for h in range(H):
            pk, pv = _exact_unit(s["prefix_pool"], s["prefix_table"][g * H + h], n_prefix[g], s)
            for b in range(s["starts"][g], s["starts"][g + 1]):
                ks, vs = [pk, s["dense_k"][b, h, :n_dense[b]].double()], [pv, s["dense_v"][b, h, :n_dense[b]].double()]
                if n_body[b]:
                    k, v = _exact_unit(s["body_pool"], s["body_table"][b * H + h], n_body[b], s)
                    ks.append(k), vs.append(v)
                p = torch.softmax(q[b, h * G:(h + 1) * G] @ torch.cat(ks).T / math.sqrt(D), -1)
                out[b, h] = p @ torch.cat(vs)
    return out.view(B, H * G, D)
