"""Prompts and shared prompts over the paged cache, as a list of measurable cases.

Three operators that a prompt goes through:

  prompt   causal attention of packed prompts of different lengths, grouped heads: row i of sequence b sees its
           keys j <= i + ctx_len[b] - q_len[b]; o = softmax(q k^T / sqrt(D)) v
  shared   the same attention over a paged cache, for a batch whose sequences share their first pages by groups
           (a system prompt): decode, verify and extension rows
  pages    what moves pages between sequences, in all layers at once: copy, fork (a sequence takes over
           another's first tokens: full pages are shared and counted, the started one is copied), compact (live
           pages move to the front of the pool)

A page holds 16 tokens of every KV head; a K (or bf16 V) block of a head is [D / 64][16 tokens][64 dims] with 8-dim
chunk j of token r at chunk position j ^ (r & 7); an E4M3 V block is [16 tokens][D] codes with one scale a token.

``own = False`` runs elementary torch operations in 32 bits; ``own = True`` calls specdec_b200.kernels.ops.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

PAGE = 16
_PACKAGE = str(Path(__file__).resolve().parents[1] / "specdec-context-scaling_b200")
_own_modules = None


def _own():
    global _own_modules
    if _own_modules is None:
        if _PACKAGE not in sys.path:
            sys.path.insert(0, _PACKAGE)
        from specdec_b200.engine.paged_cache import PagedKVCache
        from specdec_b200.kernels import ops

        _own_modules = ops, PagedKVCache
    return _own_modules


# ------------------------------------------------------------------------------------ cases
def _prompt(name, seqs, longest, shortest, heads, kv, dim, before=0, spread=0):
    """Prompts of shortest .. longest new tokens, each after ``before`` tokens whose keys are there already."""
    return {"name": name, "op": "prompt", "seqs": seqs, "longest": longest, "shortest": shortest, "heads": heads,
            "kv": kv, "dim": dim, "before": before, "spread": spread}


def _shared(name, seqs, groups, prefix, suffix, q, heads, kv, dim, v8=False, ragged=False, spread=0):
    """Sequence b in group b % groups (the last sequence alone where ragged), 0 .. suffix own tokens, q new ones."""
    return {"name": name, "op": "shared", "seqs": seqs, "groups": groups, "prefix": prefix, "suffix": suffix, "q": q,
            "heads": heads, "kv": kv, "dim": dim, "v8": v8, "ragged": ragged, "spread": spread}


def _pages(name, op, layers, kv, dim, pages, tokens=0, forks=0, moved=0, spread=0):
    return {"name": name, "op": op, "layers": layers, "kv": kv, "dim": dim, "pages": pages, "tokens": tokens,
            "forks": forks, "moved": moved, "spread": spread}


def listed():
    return [
        # one short question, target heads: the latency end
        _prompt("prompt_one_short", 1, 37, 37, 12, 2, 128),
        # a batch of questions of different lengths, draft heads
        _prompt("prompt_packed_draft", 11, 2047, 96, 14, 2, 64, spread=1),
        # the last 512 tokens of an 8192-token prompt that is read in pieces
        _prompt("prompt_chunk_512", 1, 512, 512, 12, 2, 128, before=7680),
        # four 8192-token prompts, target heads: the compute end
        _prompt("prompt_four_8k", 4, 8192, 8192, 12, 2, 128),
        # four short chats after one system prompt, a decode step: the latency end
        _shared("shared_decode_4", 4, 1, 512, 40, 1, 12, 2, 128),
        # a verify step of 64 sequences that share an 8192-token document
        _shared("shared_verify_64", 64, 1, 8192, 1024, 5, 12, 2, 128),
        # a draft decode step of 256 sequences under one system prompt
        _shared("shared_draft_decode_256", 256, 1, 4096, 512, 1, 14, 2, 64),
        # three system prompts and a sequence without one, E4M3 V, decode and verify rows mixed
        _shared("shared_groups_e4m3", 49, 3, 4000, 300, 5, 12, 2, 128, v8=True, ragged=True, spread=2),
        # a 300-token prompt forked to four sequences (two target layers' worth of a small pool)
        _pages("fork_4", "fork", 2, 2, 128, 64, tokens=300, forks=4),
        # an 8191-token prompt forked to 64 sequences, all target layers
        _pages("fork_64", "fork", 28, 2, 128, 768, tokens=8191, forks=64),
        # 512 of 1500 pages copied to others, all draft layers
        _pages("copy_512", "copy", 24, 2, 64, 1500, moved=512),
        # a target pool of 1800 pages, half of them free here and there, made dense
        _pages("compact_1800", "compact", 28, 2, 128, 1800, moved=900),
    ]


_HEADS = [(12, 2, 128), (12, 2, 128), (14, 2, 64), (14, 2, 64), (8, 8, 64), (16, 4, 128), (5, 1, 128), (24, 8, 64)]
_MOST_PAIRS = 4 * 12 * 8192 * 8193 // 2 * 128  # visible (row, key) pairs x heads x dim of prompt_four_8k
_MOST_SCORES = 4 * 12 * 8192 * 8192
_MOST_MOVED = 28 * 2 * 128 * 900  # layers x kv x dim x pages of compact_1800


def _size(rng, low, high):
    """Log-uniform over [low, high]."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "shared", "shared", "pages"])
    spread = rng.randrange(1 << 30)
    if op == "prompt":
        heads, kv, dim = rng.choice(_HEADS)
        while True:
            seqs = _size(rng, 1, 32)
            longest = _size(rng, 1, 8192)
            shortest = rng.choice([longest, max(1, longest // 10), 1])
            before = rng.choice([0, 0, _size(rng, 1, 8192)])
            c = _prompt("", seqs, longest, shortest, heads, kv, dim, before, spread)
            if (work(c)["flops"] <= 4 * _MOST_PAIRS and seqs * heads * longest * (longest + before) <= _MOST_SCORES
                    and seqs * (longest + before) <= 65536):
                break
    elif op == "shared":
        heads, kv, dim = rng.choice(_HEADS)
        while True:
            seqs = _size(rng, 1, 256)
            q = rng.choice([1, 1, 5, 5, 3, 8, _size(rng, 9, 200)])
            c = _shared("", seqs, min(seqs, rng.choice([1, 1, 2, 3, 7])), _size(rng, 1, 16384), _size(rng, 1, 1024), q,
                        heads, kv, dim, dim == 128 and rng.random() < 0.4, rng.random() < 0.5, spread)
            tokens = seqs * (c["prefix"] + c["suffix"] + q)
            if tokens * kv * dim <= 64 * 9300 * 2 * 128 * 2 and tokens * heads * q <= _MOST_SCORES // 2:
                break
    else:
        kv, dim = rng.choice([(2, 128), (2, 64), (8, 64), (1, 128)])
        layers = rng.choice([1, 2, 24, 28, 5])
        most = min(1800, 2 * _MOST_MOVED // (layers * kv * dim))
        kind = rng.choice(["fork", "copy", "compact"])
        if kind == "fork":
            forks = _size(rng, 1, min(256, most // 3))
            tokens = _size(rng, 1, PAGE * (most - forks - 1))
            pages = -(-tokens // PAGE) + forks + rng.randrange(40)
            c = _pages("", kind, layers, kv, dim, pages, tokens=tokens, forks=forks, spread=spread)
        else:
            moved = _size(rng, 1, most // 2)
            c = _pages("", kind, layers, kv, dim, 2 * moved + rng.randrange(100), moved=moved, spread=spread)
    del c["name"]
    return c


# ------------------------------------------------------------------------------------ lengths
def _prompt_lengths(case):
    r = random.Random(case["spread"])
    n, low, high = case["seqs"], case["shortest"], case["longest"]
    q = [high] + [r.randint(low, high) for _ in range(n - 1)]
    return q, [case["before"] + x for x in q]


def _shared_lengths(case):
    """(group of every sequence or -1, prefix of every group, q, own tokens before the new ones)."""
    r = random.Random(case["spread"])
    n, g, q = case["seqs"], case["groups"], case["q"]
    prefix = [max(0, case["prefix"] - 37 * i) for i in range(g)]
    group = [b % g for b in range(n)]
    if case["ragged"] and n > g:
        group[-1] = -1
    qs = [r.choice([1, q, r.randint(1, q)]) if case["ragged"] else q for _ in range(n)]
    return group, prefix, qs, [r.randint(0, case["suffix"]) for _ in range(n)]


def _starts(lengths):
    out, acc = [], 0
    for x in lengths:
        out.append(acc)
        acc += x
    return out


# ------------------------------------------------------------------------------------ inputs
def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _normal(g, *shape, level=1.0):
    x = torch.empty(*shape, dtype=torch.bfloat16, device="cuda")
    return x.normal_(0.0, level, generator=g)


def _places(lengths):
    """(sequence, index in it) of every packed row."""
    n = torch.tensor(lengths)
    b = torch.repeat_interleave(torch.arange(len(lengths)), n)
    i = torch.arange(int(n.sum())) - torch.tensor(_starts(lengths))[b]
    return b.cuda(), i.cuda()


def _prepare_prompt(case, g, s):
    q, ctx = _prompt_lengths(case)
    rows, keys, dim = sum(q), sum(ctx), case["dim"]
    # one fused projection's worth of rows; q a little larger than unit, so that a row looks at some keys more
    s["q"] = _normal(g, rows, case["heads"], dim, level=1.5)
    s["k"], s["v"] = _normal(g, keys, case["kv"], dim), _normal(g, keys, case["kv"], dim)
    s["row0"], s["kv_row0"], s["q_len"], s["ctx_len"] = _i32(_starts(q)), _i32(_starts(ctx)), _i32(q), _i32(ctx)
    s["bounds"] = (len(q), max(q), rows, max(ctx))
    s["place"] = _places(q)


def _prepare_shared(case, g, s):
    group, prefix, q, own_tokens = _shared_lengths(case)
    dim, kv, n = case["dim"], case["kv"], case["seqs"]
    full = [p // PAGE for p in prefix]  # pages that a group's sequences share
    before = [(prefix[k] if k >= 0 else 0) + t for k, t in zip(group, own_tokens)]
    ctx = [a + b for a, b in zip(before, q)]
    width = -(-max(ctx) // PAGE)
    shared = sum(full)
    own_pages = [-(-c // PAGE) - (full[k] if k >= 0 else 0) for c, k in zip(ctx, group)]
    total = shared + sum(own_pages) + 7
    order = torch.randperm(total, generator=torch.Generator().manual_seed(case["spread"])).to(torch.int32)
    table = torch.zeros(n, width, dtype=torch.int32)
    first, at = _starts(full), shared
    for b in range(n):
        lead = full[group[b]] if group[b] >= 0 else 0
        if lead:
            table[b, :lead] = order[first[group[b]]:first[group[b]] + lead]
        table[b, lead:lead + own_pages[b]] = order[at:at + own_pages[b]]
        at += own_pages[b]
    s["table"] = table.cuda()
    s["k"] = _normal(g, total, kv, PAGE * dim)
    if case["v8"]:
        x = torch.randn(total, kv, PAGE * dim, device="cuda", generator=g).mul_(100.0).clamp_(-448.0, 448.0)
        s["v"] = x.to(torch.float8_e4m3fn).view(torch.uint8)
        s["v_scale"] = torch.rand(total, kv, PAGE, device="cuda", generator=g).add_(0.5).mul_(0.01)
    else:
        s["v"], s["v_scale"] = _normal(g, total, kv, PAGE * dim), None
    s["q"] = _normal(g, sum(q), case["heads"], dim, level=1.5)
    s["row0"], s["q_len"], s["ctx_len"] = _i32(_starts(q)), _i32(q), _i32(ctx)
    s["bounds"] = (n, max(q), sum(q), max(ctx))
    members = [[b for b in range(n) if group[b] == k] for k in range(case["groups"])]
    s["members"] = _i32([b for m in members for b in m])
    s["group_start"] = _i32(_starts([len(m) for m in members]) + [sum(len(m) for m in members)])
    s["prefix_len"] = _i32(prefix)
    s["place"] = _places(q)


def _prepare_pages(case, g, s):
    r = random.Random(case["spread"])
    layers, kv, dim, pages = case["layers"], case["kv"], case["dim"], case["pages"]
    s["k"], s["v"] = _normal(g, layers, pages, kv, PAGE * dim), _normal(g, layers, pages, kv, PAGE * dim)
    order = list(range(pages))
    r.shuffle(order)
    if case["op"] == "copy":
        s["src"], s["dst"] = _i32(order[:case["moved"]]), _i32(order[case["moved"]:2 * case["moved"]])
        s["table"], s["lengths"] = s["src"].view(1, -1), _i32([PAGE * case["moved"]])
        return
    refs = torch.zeros(pages, dtype=torch.int32)
    if case["op"] == "fork":
        used = -(-case["tokens"] // PAGE)
        table = torch.full((1 + case["forks"], used + 2), -1, dtype=torch.int32)
        table[0, :used] = torch.tensor(order[:used])
        refs[order[:used]] = 1
        lengths = torch.zeros(1 + case["forks"], dtype=torch.int32)
        lengths[0] = case["tokens"]
        s["src"] = torch.zeros(case["forks"], dtype=torch.int32, device="cuda")
        s["dst"] = _i32(range(1, 1 + case["forks"]))
        s["length"] = torch.full((case["forks"],), case["tokens"], dtype=torch.int32, device="cuda")
    else:
        # live pages: sequences of up to 64 pages of their own after 8 pages that all of them share
        live = order[:case["moved"]]
        lead = live[:min(8, len(live) - 1)] if len(live) > 1 else []
        rest = live[len(lead):]
        rows = [rest[i:i + 64] for i in range(0, len(rest), 64)]
        table = torch.full((len(rows), 72 + 4), -1, dtype=torch.int32)
        for b, row in enumerate(rows):
            table[b, :len(lead) + len(row)] = torch.tensor(lead + row)
            refs[lead + row] += 1
        lengths = (table >= 0).sum(1).mul(PAGE).to(torch.int32)
        s["table0"], s["refs0"] = table.cuda(), refs.cuda()
    s["table"], s["refs"], s["lengths"] = table.cuda(), refs.cuda(), lengths.cuda()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    s = dict(case)
    if case["op"] == "prompt":
        _prepare_prompt(case, g, s)
    elif case["op"] == "shared":
        _prepare_shared(case, g, s)
    else:
        _prepare_pages(case, g, s)
    return s


# ------------------------------------------------------------------------------------ one pass, plain
def _attend(q, k, v, q_len, ctx_len, dim):
    """q (B, Q, H, D), k and v (B, KV, T, D) in fp32 -> (B, Q, H, D); rows past q_len mean nothing."""
    n, most, heads, _ = q.shape
    kv, keys = k.shape[1], k.shape[2]
    q = q.view(n, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, -1, dim)
    p = torch.matmul(q, k.transpose(2, 3)).view(n, heads, most, keys)
    last = torch.arange(most, device=q.device) + (ctx_len - q_len).long().unsqueeze(1)  # (B, Q): last visible key
    hidden = torch.arange(keys, device=q.device) > last.unsqueeze(2)
    p.mul_(1.0 / math.sqrt(dim)).masked_fill_(hidden.unsqueeze(1), float("-inf"))
    p.sub_(p.amax(dim=3, keepdim=True)).exp_()
    total = p.sum(dim=3, keepdim=True)
    o = torch.matmul(p.view(n, kv, -1, keys), v).view(n, heads, most, dim)
    return (o / total).transpose(1, 2)


def _padded(rows, row0, length, most):
    """(B, most) row numbers of packed rows; those past a sequence's length repeat its last."""
    i = torch.arange(most, device=rows.device).unsqueeze(0)
    return row0.long().unsqueeze(1) + torch.minimum(i, (length.long() - 1).clamp(min=0).unsqueeze(1))


def _plain_prompt(s):
    _, most, _, keys = s["bounds"]
    q = s["q"].float()[_padded(s["q"], s["row0"], s["q_len"], most)]
    at = _padded(s["k"], s["kv_row0"], s["ctx_len"], keys)
    k, v = s["k"].float()[at].transpose(1, 2), s["v"].float()[at].transpose(1, 2)
    return _attend(q, k, v, s["q_len"], s["ctx_len"], s["dim"])[s["place"]].to(torch.bfloat16)


def _unswizzled(blocks, dim):
    """(..., 16 * D) blocks of a bf16 pool -> (..., 16, D) rows in fp32."""
    r = torch.arange(PAGE, device=blocks.device).unsqueeze(1)
    d = torch.arange(dim, device=blocks.device)
    at = d // 64 * 1024 + r * 64 + ((d % 64 // 8) ^ (r & 7)) * 8 + d % 8
    return blocks.float()[..., at]


def _plain_shared(s):
    dim, table = s["dim"], s["table"].long()
    n, most, _, _ = s["bounds"]
    k = _unswizzled(s["k"][table], dim)  # (B, pages, KV, 16, D)
    if s["v8"]:
        v = s["v"][table].view(torch.float8_e4m3fn).float().unflatten(3, (PAGE, dim)) * s["v_scale"][table].unsqueeze(4)
    else:
        v = _unswizzled(s["v"][table], dim)
    k, v = (x.transpose(1, 2).reshape(n, s["kv"], -1, dim) for x in (k, v))
    q = s["q"].float()[_padded(s["q"], s["row0"], s["q_len"], most)]
    return _attend(q, k, v, s["q_len"], s["ctx_len"], dim)[s["place"]].to(torch.bfloat16)


def _plain_copy(s):
    src, dst = s["src"].long(), s["dst"].long()
    s["k"][:, dst] = s["k"][:, src]
    s["v"][:, dst] = s["v"][:, src]
    return s["k"], s["v"]


def _plain_fork(s):
    table, refs = s["table"], s["refs"]
    src, dst, length = s["src"].long(), s["dst"].long(), s["length"].long()
    old = table[dst]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).flatten().int())
    full, started = length // PAGE, length % PAGE > 0
    column = torch.arange(table.shape[1], device=table.device)
    rows = torch.where(column < full.unsqueeze(1), table[src], -1)
    refs.index_add_(0, rows.clamp(min=0).flatten().long(), (rows >= 0).flatten().int())
    free = torch.argsort((refs > 0).int(), stable=True)  # free pages first, the lowest first
    new = free[(started.long().cumsum(0) - 1).clamp(min=0)]
    refs.index_add_(0, new, started.int())
    here = (column == full.unsqueeze(1)) & started.unsqueeze(1)
    from_page, to_page = table[src, full][started].long(), new[started]
    s["k"][:, to_page] = s["k"][:, from_page]
    s["v"][:, to_page] = s["v"][:, from_page]
    table[dst] = torch.where(here, new.unsqueeze(1).int(), rows)
    s["lengths"][dst] = length.int()
    return s["k"], s["v"], table, refs, s["lengths"]


def _plain_compact(s):
    table, refs = s["table"].copy_(s["table0"]), s["refs"].copy_(s["refs0"])
    live = refs > 0
    n_live = live.sum()
    page = torch.arange(refs.numel(), device=refs.device)
    from_page, to_page = page[live & (page >= n_live)], page[~live & (page < n_live)]
    s["k"][:, to_page] = s["k"][:, from_page]
    s["v"][:, to_page] = s["v"][:, from_page]
    place = page.int()
    place[from_page] = to_page.int()
    table.copy_(torch.where(table >= 0, place[table.clamp(min=0).long()], -1))
    refs[to_page] = refs[from_page]
    refs[from_page] = 0
    return s["k"], s["v"], table, refs, n_live.int()


# ------------------------------------------------------------------------------------ one pass, the framework's
def _batch(s):
    ops, _ = _own()
    n, most, rows, keys = s["bounds"]
    return ops.RaggedBatch(s["row0"], s["q_len"], s["ctx_len"], n, most, rows, keys)


def _cache(s):
    """The cache object that a program keeps around its pools."""
    if "cache" not in s:
        _, cache = _own()
        if s["op"] == "shared":
            s["cache"] = cache.from_pools([s["k"]], [s["v"]], [s["v_scale"]] if s["v8"] else None, s["table"],
                                          s["ctx_len"], s["dim"])
        else:
            s["cache"] = cache.from_pools(list(s["k"]), list(s["v"]), None, s["table"], s["lengths"], s["dim"],
                                          page_refs=s.get("refs"))
    return s["cache"]


def _own_pass(s):
    ops, _ = _own()
    op = s["op"]
    if op == "prompt":
        return ops.prompt_attention(s["q"], s["k"], s["v"], _batch(s), kv_row0=s["kv_row0"])
    cache = _cache(s)
    if op == "shared":
        prefix = ops.SharedPrefix(s["group_start"], s["members"], s["prefix_len"], s["groups"], s["members"].numel())
        return ops.shared_prefix_attention(s["q"], cache, 0, _batch(s), prefix)
    if op == "copy":
        ops.copy_pages(cache, s["src"], s["dst"])
        return s["k"], s["v"]
    if op == "fork":
        ops.fork_sequences(cache, s["src"], s["dst"], s["length"])
        return s["k"], s["v"], s["table"], s["refs"], s["lengths"]
    s["table"].copy_(s["table0"])
    s["refs"].copy_(s["refs0"])
    return s["k"], s["v"], s["table"], s["refs"], ops.compact_pages(cache)


_PLAIN = {"prompt": _plain_prompt, "shared": _plain_shared, "copy": _plain_copy, "fork": _plain_fork,
          "compact": _plain_compact}


def run(state):
    """One pass.  Compacting starts from the same scattered pages each time (two small copies put the table and
    the counts back; what a pass moves away stays readable where it was)."""
    return _own_pass(state) if own else _PLAIN[state["op"]](state)


# ------------------------------------------------------------------------------------ accounting
def work(case):
    op, kv, dim = case["op"], case["kv"], case["dim"]
    if op == "prompt":
        q, ctx = _prompt_lengths(case)
        pairs = sum(n * (c - n) + n * (n + 1) // 2 for n, c in zip(q, ctx))
        return {"bytes": 4 * sum(q) * case["heads"] * dim + 4 * sum(ctx) * kv * dim,
                "flops": 4 * dim * case["heads"] * pairs}
    if op == "shared":
        group, prefix, q, own_tokens = _shared_lengths(case)
        before = [(prefix[k] if k >= 0 else 0) + t for k, t in zip(group, own_tokens)]
        pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(q, before))
        read = sum(p // PAGE * PAGE for p in prefix)  # tokens of the pages that are read, shared ones once
        read += sum(c + n - (prefix[k] // PAGE * PAGE if k >= 0 else 0) for n, c, k in zip(q, before, group))
        token = kv * (2 * dim + (dim + 4 if case["v8"] else 2 * dim))
        return {"bytes": read * token + 4 * sum(q) * case["heads"] * dim, "flops": 4 * dim * case["heads"] * pairs}
    page = case["layers"] * kv * PAGE * dim * 4  # K and V
    if op == "copy":
        return {"bytes": 2 * case["moved"] * page, "flops": 0}
    if op == "fork":
        used, started = -(-case["tokens"] // PAGE), case["tokens"] % PAGE > 0
        return {"bytes": ((1 + case["forks"]) * page if started else 0) + 4 * used * (1 + case["forks"]), "flops": 0}
    # pages of the upper part that are live move; about half of the live ones where half of the pool is free
    r = random.Random(case["spread"])
    order = list(range(case["pages"]))
    r.shuffle(order)
    moves = sum(p >= case["moved"] for p in order[:case["moved"]])
    return {"bytes": 2 * moves * page + 8 * case["pages"], "flops": 0}


# ------------------------------------------------------------------------------------ 64 bits
def _exact_rows(q, k, v, first):
    """q (Q, H, D), k and v (T, KV, D) of one sequence in fp64; row i sees keys 0 .. first + i."""
    rows, heads, dim = q.shape
    kv = k.shape[1]
    out = torch.empty_like(q)
    see = torch.ones(rows, k.shape[0], dtype=torch.bool, device=q.device).tril_(first)
    for h in range(heads):
        e = torch.einsum("id,jd->ij", q[:, h], k[:, h * kv // heads]) / dim ** 0.5
        e = torch.softmax(torch.where(see, e, -math.inf), dim=1)
        out[:, h] = e @ v[:, h * kv // heads]
    return out


def _exact_pages(case, s):
    """Python integers for the tables; the pools' values with the copied pages in their places."""
    k, v = s["k"].double(), s["v"].double()
    if case["op"] == "copy":
        moves = list(zip(s["src"].tolist(), s["dst"].tolist()))
        rest = ()
    elif case["op"] == "fork":
        table, refs, lengths = s["table"].tolist(), s["refs"].tolist(), s["lengths"].tolist()
        moves = []
        for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), s["length"].tolist()):
            for j in range(n // PAGE):
                table[b][j] = table[a][j]
                refs[table[a][j]] += 1
            lengths[b] = n
        for a, b, n in zip(s["src"].tolist(), s["dst"].tolist(), s["length"].tolist()):
            if n % PAGE:
                page = refs.index(0)
                refs[page] = 1
                table[b][n // PAGE] = page
                moves.append((table[a][n // PAGE], page))
        rest = (table, refs, lengths)
    else:
        table, refs = s["table0"].tolist(), s["refs0"].tolist()
        n_live = sum(c > 0 for c in refs)
        moves = list(zip((p for p in range(n_live, len(refs)) if refs[p]), (p for p in range(n_live) if not refs[p])))
        to = dict(moves)
        for a, b in moves:
            refs[a], refs[b] = 0, refs[a]
        rest = ([[to.get(p, p) for p in row] for row in table], refs, n_live)
    for a, b in moves:
        k[:, b], v[:, b] = s["k"][:, a].double(), s["v"][:, a].double()
    return (k, v) + tuple(torch.tensor(x, dtype=torch.int32, device="cuda") for x in rest)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] not in ("prompt", "shared"):
        return _exact_pages(case, s)
    out = []
    dim, kv = case["dim"], case["kv"]
    if case["op"] == "prompt":
        q_lens, ctx = _prompt_lengths(case)
        for a, n, b, c in zip(_starts(q_lens), q_lens, _starts(ctx), ctx):
            out.append(_exact_rows(s["q"][a:a + n].double(), s["k"][b:b + c].double(), s["v"][b:b + c].double(), c - n))
        return torch.cat(out)
    token = torch.arange(PAGE)
    chunks = torch.stack([torch.stack([(torch.arange(8) ^ (int(t) & 7)) + 8 * int(t) for t in token])
                          + 128 * half for half in range(dim // 64)], 1).reshape(PAGE, dim // 8).cuda()
    for b, (a, n, c) in enumerate(zip(s["row0"].tolist(), s["q_len"].tolist(), s["ctx_len"].tolist())):
        pages = s["table"][b, :-(-c // PAGE)].long()

        def rows_of(pool):  # a block as chunks of 8 dims, each token's chunks in order
            x = pool[pages].double().unflatten(2, (-1, 8))[:, :, chunks]  # (pages, KV, 16, D / 8, 8)
            return x.flatten(3).transpose(1, 2).reshape(-1, kv, dim)[:c]

        if case["v8"]:
            x = s["v"][pages].view(torch.float8_e4m3fn).double().unflatten(2, (PAGE, dim))
            v = (x * s["v_scale"][pages].double().unsqueeze(3)).transpose(1, 2).reshape(-1, kv, dim)[:c]
        else:
            v = rows_of(s["v"])
        out.append(_exact_rows(s["q"][a:a + n].double(), rows_of(s["k"]), v, c - n))
    return torch.cat(out)
