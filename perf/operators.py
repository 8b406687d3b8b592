"""Measured cases of the attention operators without a cache and over draft trees, and of the cache's page operators.

Five operators, each as one pass of a serving program:

* ``prompt`` -- ``prompt_attention``: packed sequences with plain K/V rows, causal or bidirectional;
* ``tree`` -- ``paged_tree_attention``: drafted tokens that form a tree, over a paged cache;
* ``copy`` -- ``kv_pages.copy_pages``: whole pages duplicated in every layer;
* ``fork`` -- ``kv_pages.free_sequences`` then ``kv_pages.fork_sequences``: one step of a search that
  drops its branches and opens new ones;
* ``keep`` -- ``kv_pages.keep_accepted_tokens``: the accepted path of a verified draft moved together.

With ``own`` false ``run`` computes the plain form in elementary torch operations, else it calls this package.
"""

import math
import os
import random
import sys

import torch

own = False

_HERE = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_SCORES = 1 << 30  # scores that the plain form holds at once (4 GB in fp32)


def _package():
    path = os.path.join(_HERE, "minicpm-attention-optimization-iluvatar_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import minicpm_b200

    return minicpm_b200


# --------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # A few short user turns that arrive together: launch latency and ragged, odd lengths.
        dict(name="prompt short", op="prompt", seqs=4, min_len=17, max_len=131, prefix=0, hq=16, hkv=2, dim=128,
             dtype="bf16", causal=True, lens_seed=1),
        # An encoder or embedding batch: every token sees its whole sequence, one KV head per query head.
        dict(name="prompt encoder", op="prompt", seqs=33, min_len=60, max_len=517, prefix=0, hq=12, hkv=12, dim=64,
             dtype="fp16", causal=False, lens_seed=2),
        # Long documents, the first pass of a model with 16 query and 2 KV heads.
        dict(name="prompt 16k", op="prompt", seqs=4, min_len=8192, max_len=16384, prefix=0, hq=16, hkv=2, dim=128,
             dtype="bf16", causal=True, lens_seed=3),
        # One user, a small draft: the latency of one verification step.
        dict(name="tree one user", op="tree", seqs=1, min_len=4000, max_len=4096, nodes=16, ragged=False, page=16,
             hq=16, hkv=2, dim=128, dtype="bf16", lens_seed=4),
        # Ragged drafts of small models with wide heads groups, odd lengths, larger pages.
        dict(name="tree ragged", op="tree", seqs=7, min_len=33, max_len=2047, nodes=61, ragged=True, page=32,
             hq=32, hkv=8, dim=64, dtype="fp16", lens_seed=5),
        # A full serving batch at long context, each sequence with a draft of 32 nodes.
        dict(name="tree batch 16k", op="tree", seqs=64, min_len=8192, max_len=16384, nodes=32, ragged=False, page=16,
             hq=16, hkv=2, dim=128, dtype="bf16", lens_seed=6),
        # A handful of prefix pages duplicated before they are written to.
        dict(name="copy few", op="copy", pages=5, pool=256, layers=8, page=16, hkv=2, dim=128, dtype="bf16"),
        # A long prefix duplicated in a deep model.
        dict(name="copy prefix", op="copy", pages=509, pool=2048, layers=32, page=16, hkv=2, dim=128, dtype="bf16"),
        # Parallel sampling: one prompt answered several times.
        dict(name="fork samples", op="fork", parents=1, fanout=5, min_len=300, max_len=300, pool=512, layers=8, page=16,
             hkv=2, dim=128, dtype="bf16", lens_seed=9),
        # A beam search over a full batch with long contexts.
        dict(name="fork beams", op="fork", parents=32, fanout=4, min_len=1024, max_len=4096, pool=8192, layers=8,
             page=16, hkv=2, dim=128, dtype="bf16", lens_seed=10),
        # One user: the accepted nodes of a small draft.
        dict(name="keep one user", op="keep", seqs=1, min_len=1000, max_len=1000, nodes=16, most=5, layers=8, page=16,
             hkv=2, dim=128, dtype="bf16", lens_seed=11),
        # A full batch in a deep model.
        dict(name="keep batch", op="keep", seqs=64, min_len=200, max_len=700, nodes=32, most=9, layers=32, page=16,
             hkv=2, dim=128, dtype="bf16", lens_seed=12),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prompt", "prompt", "tree", "tree", "copy", "fork", "keep"])
    dim = rng.choice([64, 128, 128, 256])
    hkv, group = rng.choice([(2, 8), (8, 4), (1, 16), (4, 1), (2, 6), (12, 1)])
    base = dict(op=op, dtype=rng.choice(["bf16", "fp16"]), lens_seed=rng.randrange(1 << 20))
    heads = dict(hq=hkv * group, hkv=hkv, dim=dim)
    page = rng.choice([16, 32, 64])
    if op == "prompt":
        longest = _log_int(rng, 1, 8192)
        seqs, prefix = _log_int(rng, 1, 64), rng.choice([0, 0, _log_int(rng, 1, 2048)])
        while seqs > 1 and seqs * longest * (longest + prefix) * heads["hq"] * dim > 2 ** 39:
            seqs //= 2
        return dict(base, **heads, seqs=seqs, min_len=max(1, longest // rng.choice([1, 2, 8])), max_len=longest,
                    prefix=prefix, causal=rng.random() < 0.7)
    if op == "tree":
        longest = _log_int(rng, 2, 32768)
        nodes = _log_int(rng, 1, 128)
        seqs = _log_int(rng, 1, 64)
        while seqs > 1 and (seqs * longest * hkv * dim > 2 ** 28 or seqs * longest * nodes * heads["hq"] * dim > 2 ** 36):
            seqs //= 2
        return dict(base, **heads, seqs=seqs, min_len=max(1, longest // rng.choice([1, 2, 8])), max_len=longest,
                    nodes=nodes, ragged=rng.random() < 0.5, page=page)
    rows = dict(hkv=hkv, dim=dim, page=page)
    layers = _log_int(rng, 1, 32)
    budget = 2 ** 28 // (layers * page * hkv * dim)  # pages that a pool of at most 1 GB holds
    if op == "copy":
        pool = max(4, min(2048, budget))
        return dict(base, **rows, layers=layers, pool=pool, pages=_log_int(rng, 1, pool // 2))
    if op == "fork":
        parents, fanout = _log_int(rng, 1, 32), _log_int(rng, 1, 8)
        longest = max(1, min(_log_int(rng, 1, 4096), max(1, (budget - parents * fanout) // (parents + 1) - 1) * page))
        pool = parents * (-(-longest // page)) + parents * fanout + 3
        return dict(base, **rows, layers=layers, parents=parents, fanout=fanout, min_len=max(1, longest // 3),
                    max_len=longest, pool=pool)
    seqs, nodes = _log_int(rng, 1, 64), _log_int(rng, 1, 64)
    longest = _log_int(rng, 1, 512)
    while seqs > 1 and seqs * (-(-(longest + nodes) // page) + 1) > budget:
        seqs //= 2
    return dict(base, **rows, layers=layers, seqs=seqs, min_len=max(1, longest // 2), max_len=longest, nodes=nodes,
                most=rng.randint(0, nodes))


def _lens(case, key="seqs"):
    r = random.Random(case["lens_seed"])
    return [r.randint(case["min_len"], case["max_len"]) for _ in range(case[key])]


def _drafts(case):
    r = random.Random(case["lens_seed"] + 1)
    n = case["nodes"]
    return [r.randint(1, n) if case.get("ragged") else n for _ in range(case["seqs"])]


def _accepted_counts(case):
    r = random.Random(case["lens_seed"] + 2)
    return [min(n, r.randint(0, case["most"])) for n in _drafts(case)]


# ------------------------------------------------------------------------------------------- prepare
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cu(lens):
    total, out = 0, [0]
    for n in lens:
        total += n
        out.append(total)
    return _ints(out)


def _tables(rng, lens, page, pool, cols):
    """Physical pages of sequences of these lengths, a seeded permutation of the pool; -1 behind a sequence's last page."""
    ids = list(range(pool))
    rng.shuffle(ids)
    rows, at = [], 0
    for n in lens:
        need = -(-n // page)
        rows.append(ids[at:at + need] + [-1] * (cols - need))
        at += need
    return rows


def _layers(g, case, pool):
    """[layers, pool, 2 (K, V), page, hkv, dim], layer by layer so that the fp32 draws stay small."""
    shape = (pool, 2, case["page"], case["hkv"], case["dim"])
    cache = torch.empty((case["layers"],) + shape, dtype=_DTYPES[case["dtype"]], device="cuda")
    for layer in cache:
        layer.copy_(torch.randn(shape, generator=g, device="cuda", dtype=torch.float32))
    return cache


def prepare(case, seed):
    g, rng = _gen(seed), random.Random(seed)
    dtype = _DTYPES[case["dtype"]]
    s = dict(case=case, op=case["op"])
    if own:
        s["package"] = _package()
    if case["op"] == "prompt":
        ql = _lens(case)
        kl = [n + case["prefix"] for n in ql]
        d = case["dim"]
        s.update(q=_normal(g, (sum(ql), case["hq"], d), dtype), k=_normal(g, (sum(kl), case["hkv"], d), dtype),
                 v=_normal(g, (sum(kl), case["hkv"], d), dtype), cu_q=_cu(ql), cu_k=_cu(kl), ql=ql, kl=kl,
                 scale=d ** -0.5)
        s["out"] = torch.empty_like(s["q"])
        return s
    if case["op"] == "tree":
        n, d, page = _drafts(case), case["dim"], case["page"]
        kl = [c + m for c, m in zip(_lens(case), n)]
        cols = -(-max(kl) // page)
        pool = sum(-(-x // page) for x in kl) + 1
        cache = _normal(g, (pool, 2, page, case["hkv"], d), dtype)
        most = max(n)
        mask = torch.zeros(sum(n), most, dtype=torch.bool)
        row = 0
        for m in n:  # node i: its parent's ancestors and itself; a parent of -1 is the context
            for i in range(m):
                parent = rng.randint(-1, i - 1)
                if parent >= 0:
                    mask[row + i] = mask[row + parent]
                mask[row + i, i] = True
            row += m
        # A scheduler's table holds 0 behind a sequence's last page.
        table = [[max(p, 0) for p in r] for r in _tables(rng, kl, page, pool, cols)]
        s.update(q=_normal(g, (sum(n), case["hq"], d), dtype), cache=cache, table=_ints(table), mask=mask.cuda(),
                 lens=_ints(kl), cu_q=_cu(n), kl=kl, n=n, scale=d ** -0.5)
        s["out"] = torch.empty_like(s["q"])
        return s
    pool = case.get("pool") or sum(-(-(x + case["nodes"]) // case["page"]) for x in _lens(case)) + 1
    cache = _layers(g, case, pool)
    s["cache"] = cache
    if case["op"] == "copy":
        ids = list(range(pool))
        rng.shuffle(ids)
        s.update(src=_ints(ids[:case["pages"]]), dst=_ints(ids[pool - case["pages"]:]))
    elif case["op"] == "fork":
        lens = _lens(case, "parents")
        kids = case["parents"] * case["fanout"]
        cols = -(-case["max_len"] // case["page"])
        table = _tables(rng, lens, case["page"], pool, cols) + [[-1] * cols for _ in range(kids)]
        refs = [0] * pool
        for row in table:
            for p in row:
                if p >= 0:
                    refs[p] += 1
        s.update(table=_ints(table), lens=_ints(lens + [0] * kids), refs=_ints(refs),
                 parents=_ints([rng.randrange(case["parents"]) for _ in range(kids)]),
                 children=_ints(range(case["parents"], case["parents"] + kids)))
    else:
        ctx, n, acc = _lens(case), _drafts(case), _accepted_counts(case)
        kl = [c + m for c, m in zip(ctx, n)]
        table = _tables(rng, kl, case["page"], pool, -(-max(kl) // case["page"]))
        most = max(1, max(acc))
        path = [sorted(rng.sample(range(m), a)) + [-1] * (most - a) for m, a in zip(n, acc)]
        s.update(table=_ints(table), context=_ints(ctx), accepted=_ints(path), counts=_ints(acc), lens=_ints(kl))
    if own:
        s["layers"] = s["package"].kv_pages.cache_layers(list(cache))
    return s


# ----------------------------------------------------------------------------------------------- run
def run(s):
    return globals()["_" + s["op"]](s)


def _softmax_rows(x, seen):
    """exp(x - max) / sum over the last dimension where `seen`; a row that sees nothing is zero."""
    x = x.masked_fill_(~seen, float("-inf"))
    top = x.amax(dim=-1, keepdim=True)
    x = x.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    return x.div_(x.sum(dim=-1, keepdim=True).clamp_min_(1e-30))


def _prompt(s):
    case = s["case"]
    if own:
        return s["package"].prompt_attention(
            s["q"], s["k"], s["v"], s["out"], s["cu_q"], max(s["ql"]), s["scale"], causal=case["causal"],
            cu_seqlens_k=s["cu_k"], max_seqlen_k=max(s["kl"]))
    dev, d, hkv = s["q"].device, case["dim"], case["hkv"]
    group = case["hq"] // hkv
    mq, mk = max(s["ql"]), max(s["kl"])
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    step = max(1, _SCORES // (case["hq"] * mq * mk))
    for b in range(0, len(s["ql"]), step):  # as many sequences at once as their scores leave room for
        q0, q1, k0, k1 = cu_q[b:b + step], cu_q[b + 1:b + 1 + step], cu_k[b:b + step], cu_k[b + 1:b + 1 + step]
        q1, k1 = q1[:len(q0)], k1[:len(k0)]
        q0, k0 = q0[:len(q1)], k0[:len(k1)]
        i, j = torch.arange(mq, device=dev), torch.arange(mk, device=dev)
        ql, kl = (q1 - q0)[:, None], (k1 - k0)[:, None]
        row, has_q, has_k = q0[:, None] + i, i < ql, j < kl
        at_q, at_k = row.clamp_max(s["q"].shape[0] - 1), (k0[:, None] + j).clamp_max(s["k"].shape[0] - 1)
        q = s["q"][at_q].float().view(len(q0), mq, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(len(q0), hkv, group * mq, d)
        k = s["k"][at_k].float().permute(0, 2, 3, 1)
        v = s["v"][at_k].float().permute(0, 2, 1, 3)
        x = torch.matmul(q, k).mul_(s["scale"]).view(len(q0), hkv, group, mq, mk)
        seen = has_k[:, None, :].expand(-1, mq, -1)
        if case["causal"]:
            seen = seen & (j <= (kl - ql + i)[:, :, None])
        p = _softmax_rows(x, seen[:, None, None])
        o = torch.matmul(p.view(len(q0), hkv, group * mq, mk), v).view(len(q0), hkv, group, mq, d)
        s["out"][row[has_q]] = o.permute(0, 3, 1, 2, 4).reshape(len(q0), mq, case["hq"], d).to(s["out"].dtype)[has_q]
    return s["out"]


def _tree(s):
    case = s["case"]
    if own:
        return s["package"].paged_tree_attention(
            s["q"], s["cache"][:, 0], s["cache"][:, 1], s["out"], s["mask"], s["table"], s["lens"], s["cu_q"],
            max(s["n"]), max(s["kl"]), s["scale"])
    dev, d, hkv = s["q"].device, case["dim"], case["hkv"]
    group, seqs = case["hq"] // hkv, len(s["n"])
    n, mk = max(s["n"]), max(s["kl"])
    rows = s["cache"][s["table"].long()]  # [seqs, pages, 2, page, hkv, dim]
    k = rows[:, :, 0].reshape(seqs, -1, hkv, d)[:, :mk].float().permute(0, 2, 3, 1)
    v = rows[:, :, 1].reshape(seqs, -1, hkv, d)[:, :mk].float().permute(0, 2, 1, 3)
    cu = s["cu_q"].long()
    first, count = cu[:-1, None], (cu[1:] - cu[:-1])[:, None]
    i, j = torch.arange(n, device=dev), torch.arange(mk, device=dev)
    has, row = i < count, first + i
    at = row.clamp_max(s["q"].shape[0] - 1)
    lens = s["lens"].long()[:, None]
    node = j - (lens - count)  # drafted node at each key, negative in the context
    drafted = torch.gather(s["mask"][at], 2, node.clamp(0, n - 1)[:, None, :].expand(-1, n, -1))
    seen = (j < lens)[:, None] & ((node < 0)[:, None] | drafted)
    q = s["q"][at].float().view(seqs, n, hkv, group, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, group * n, d)
    x = torch.matmul(q, k).mul_(s["scale"]).view(seqs, hkv, group, n, mk)
    p = _softmax_rows(x, seen[:, None, None])
    o = torch.matmul(p.view(seqs, hkv, group * n, mk), v).view(seqs, hkv, group, n, d)
    s["out"][row[has]] = o.permute(0, 3, 1, 2, 4).reshape(seqs, n, case["hq"], d).to(s["out"].dtype)[has]
    return s["out"]


def _copy(s):
    if own:
        s["package"].kv_pages.copy_pages(s["layers"], s["src"], s["dst"])
        return s["cache"]
    s["cache"][:, s["dst"].long()] = s["cache"][:, s["src"].long()]
    return s["cache"]


def _fork(s):
    table, lens, refs, cache = s["table"], s["lens"], s["refs"], s["cache"]
    if own:
        kv = s["package"].kv_pages
        kv.free_sequences(table, lens, refs, s["children"])
        kv.fork_sequences(s["layers"], table, lens, refs, s["parents"], s["children"])
        return dict(table=table, lens=lens, refs=refs, cache=cache)
    page = cache.shape[3]
    kids, parents = s["children"].long(), s["parents"].long()
    # The children of the step before give their pages back.
    old = table[kids]
    refs.index_add_(0, old.clamp_min(0).view(-1).long(), -(old >= 0).view(-1).to(refs.dtype))
    table[kids] = -1
    lens[kids] = 0
    # Full pages are shared; a partial last page gets the lowest free page, in the order of the children.
    plens = lens[parents]
    full, tail = torch.div(plens, page, rounding_mode="floor"), plens % page
    cols = torch.arange(table.shape[1], device=table.device)
    rows = torch.where(cols < full[:, None], table[parents], torch.full_like(old, -1))
    refs.index_add_(0, rows.clamp_min(0).view(-1).long(), (rows >= 0).view(-1).to(refs.dtype))
    some = tail > 0
    fresh = torch.nonzero(refs == 0).view(-1)[:int(some.sum())]
    last = full[some].long()
    source = table[parents[some], last].long()
    rows[torch.nonzero(some).view(-1), last] = fresh.to(rows.dtype)
    refs[fresh] = 1
    table[kids] = rows
    lens[kids] = plens
    keep = (torch.arange(page, device=table.device) < tail[some][:, None]).view(1, -1, 1, page, 1, 1)
    cache[:, fresh] = torch.where(keep, cache[:, source], cache[:, fresh])
    return dict(table=table, lens=lens, refs=refs, cache=cache)


def _keep(s):
    if own:
        s["package"].kv_pages.keep_accepted_tokens(s["layers"], s["table"], s["context"], s["accepted"], s["counts"],
                                                   s["lens"])
        return dict(lens=s["lens"], cache=s["cache"])
    cache, page = s["cache"], s["cache"].shape[3]
    i = torch.arange(s["accepted"].shape[1], device=cache.device)
    some = i < s["counts"][:, None]
    to = (s["context"][:, None] + i).long()[some]
    at = (s["context"][:, None] + s["accepted"]).long()[some]
    seq = torch.arange(len(s["context"]), device=cache.device)[:, None].expand_as(some)[some]
    table = s["table"].long()
    rows = cache[:, table[seq, at // page], :, at % page]  # a copy: sources are read before any row is written
    cache[:, table[seq, to // page], :, to % page] = rows
    s["lens"].copy_(s["context"] + s["counts"])
    return dict(lens=s["lens"], cache=cache)


# ---------------------------------------------------------------------------------------------- work
def work(case):
    row = case["hkv"] * case["dim"] * 2  # bytes of one token's K (or V) row
    if case["op"] == "prompt":
        ql = _lens(case)
        kl = [n + case["prefix"] for n in ql]
        pairs = sum(q * (k - q) + q * (q + 1) // 2 if case["causal"] else q * k for q, k in zip(ql, kl))
        return dict(bytes=2 * sum(kl) * row + 2 * sum(ql) * case["hq"] * case["dim"] * 2,
                    flops=4 * pairs * case["hq"] * case["dim"])
    if case["op"] == "tree":
        ctx, n = _lens(case), _drafts(case)
        return dict(bytes=2 * (sum(ctx) + sum(n)) * row + 2 * sum(n) * case["hq"] * case["dim"] * 2 + sum(n) * max(n),
                    flops=4 * sum(m * (c + 1) for c, m in zip(ctx, n)) * case["hq"] * case["dim"])
    token = 2 * row * case["layers"]  # K and V of one token in every layer
    if case["op"] == "copy":
        return dict(bytes=2 * case["pages"] * case["page"] * token, flops=0)
    if case["op"] == "fork":
        # A child's tail depends on the parent that it draws: the mean over the parents stands for it.
        lens = _lens(case, "parents")
        kids = case["parents"] * case["fanout"]
        pages = sum(-(-n // case["page"]) for n in lens) / len(lens)
        tail = sum(n % case["page"] for n in lens) / len(lens)
        return dict(bytes=kids * (2 * tail * token + 2 * pages * 8), flops=0)
    return dict(bytes=2 * sum(_accepted_counts(case)) * token + case["seqs"] * 16, flops=0)


# --------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions, one sequence (or page) after the other, in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "prompt":
        return _exact_attention(s, [(b, q, k) for b, (q, k) in enumerate(zip(s["ql"], s["kl"]))], _rows_of_prompt)
    if case["op"] == "tree":
        return _exact_attention(s, [(b, q, k) for b, (q, k) in enumerate(zip(s["n"], s["kl"]))], _rows_of_tree)
    if case["op"] == "copy":
        want = s["cache"].double()
        src, dst = s["src"].tolist(), s["dst"].tolist()
        taken = want[:, src].clone()
        for n, p in enumerate(dst):
            want[:, p] = taken[:, n]
        return want
    if case["op"] == "fork":
        page, cache = case["page"], s["cache"].double()
        table, lens, refs = s["table"].tolist(), s["lens"].tolist(), s["refs"].tolist()
        first = [x[:] for x in table]
        for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
            for col in range(lens[p] // page):
                table[c][col] = first[p][col]
                refs[first[p][col]] += 1
        for p, c in zip(s["parents"].tolist(), s["children"].tolist()):
            used = lens[p] % page
            if used:
                new = refs.index(0)
                refs[new] = 1
                table[c][lens[p] // page] = new
                cache[:, new, :, :used] = cache[:, first[p][lens[p] // page], :, :used]
            lens[c] = lens[p]
        return dict(table=_ints(table), lens=_ints(lens), refs=_ints(refs), cache=cache)
    cache, table = s["cache"].double(), s["table"].tolist()
    context, page = s["context"].tolist(), case["page"]
    for b, path in enumerate(s["accepted"].tolist()):
        for i, node in enumerate(path[:int(s["counts"][b])]):
            a, t = context[b] + node, context[b] + i
            cache[:, table[b][t // page], :, t % page] = cache[:, table[b][a // page], :, a % page].clone()
    return dict(lens=s["context"] + s["counts"], cache=cache)


def _rows_of_prompt(s, b, q, k):
    k0 = int(s["cu_k"][b])
    i, j = torch.arange(q, device="cuda")[:, None], torch.arange(k, device="cuda")
    seen = (j - i <= k - q) if s["case"]["causal"] else torch.ones(q, k, dtype=torch.bool, device="cuda")
    return s["k"][k0:k0 + k], s["v"][k0:k0 + k], seen


def _rows_of_tree(s, b, q, k):
    page, row = s["case"]["page"], int(s["cu_q"][b])
    pages = s["table"][b, :-(-k // page)].long()
    rows = s["cache"].index_select(0, pages).transpose(0, 1).flatten(1, 2)[:, :k]
    seen = torch.ones(q, k, dtype=torch.bool, device="cuda")
    seen[:, k - q:] = s["mask"][row:row + q, :q]
    return rows[0], rows[1], seen


def _exact_attention(s, seqs, rows_of):
    case = s["case"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    group = case["hq"] // case["hkv"]
    for b, q, k in seqs:
        keys, values, seen = rows_of(s, b, q, k)
        r0 = int(s["cu_q"][b])
        for h in range(case["hq"]):
            kh, vh = keys[:, h // group].double(), values[:, h // group].double()
            step = max(1, (1 << 28) // k)
            for r in range(0, q, step):
                see = seen[r:r + step]
                x = (s["q"][r0 + r:min(r0 + r + step, r0 + q), h].double() @ kh.T) * s["scale"]
                x = torch.where(see, x, torch.full_like(x, -math.inf))
                w = torch.exp(x - x.max(dim=1, keepdim=True).values.clamp_min(-1e300))
                total = w.sum(dim=1, keepdim=True)
                out[r0 + r:r0 + r + x.shape[0], h] = torch.where(total > 0, (w @ vh) / total.clamp_min(1e-300), 0.0)
    return out
