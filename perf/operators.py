"""Work of the dense side of interattn_b200, as measurable cases: many answers to one prompt over the paged cache.

Three operators, through their public entry points:

* ``prompt``  causal attention over whole prompts packed one after the other, ``dense_attention.PromptAttention.run``;
              with ``prior`` tokens in the cache already it is the continuation of a prompt.
* ``shared``  one decode step (single tokens) of sequences that share the pages of a long prefix in groups,
              ``dense_attention.SharedPrefixAttention.step``.
* ``pages``   the pages behind both, ``page_cache.PageCache``: ``admit`` (free rows, give them pages for new prompts, write
              every layer's keys and values), ``fork`` (free rows, make them children of running sequences) and
              ``compact`` (close the holes that freed sequences left).

With ``own`` false everything is computed by elementary torch operations in fp32 (whole-number bookkeeping for the pages).

Data: seeded N(0, 1) queries, keys and values, the key channels scaled by a log-normal(0, 0.5) factor (key outliers); pages
are random permutations of the pool; lengths are uniform draws between a case's bounds.
"""

import math
import random
import types

import torch

own = False

PAGE = 16
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}

# Attention geometries (query heads, kv heads, head_dim): Llama-3-8B and -70B, the fp32 configuration that also runs on a CPU,
# the decoder's "tiny" preset, and for the drawn cases heads of their own, odd groups and one kv head for all.
L8B = {"dtype": "bf16", "q_heads": 32, "kv_heads": 8, "head_dim": 128}
L70B = {"dtype": "bf16", "q_heads": 64, "kv_heads": 8, "head_dim": 128}
SMALL_F32 = {"dtype": "f32", "q_heads": 8, "kv_heads": 2, "head_dim": 64}
TINY = {"dtype": "bf16", "q_heads": 8, "kv_heads": 2, "head_dim": 64}
DRAWN = [(32, 8, 128), (64, 8, 128), (32, 8, 64), (8, 2, 64), (12, 4, 128), (16, 16, 64), (8, 8, 128), (16, 1, 128), (14, 2, 64)]


def listed():
    return [
        # Four short prompts in fp32: all latency, one of them a single token.
        dict(SMALL_F32, kind="prompt", name="prompt_f32_small", lens="1,130,37,64", prior="0,0,0,0"),
        # A batch of chat turns at the Llama-3-8B geometry, a few to a thousand tokens each.
        dict(L8B, kind="prompt", name="prompt_8b_chat", lens=_uniform(32, 17, 1024, 1), prior=_text([0] * 32)),
        # The next pieces of half-read documents, small heads: few queries after many keys.
        dict(TINY, kind="prompt", name="prompt_d64_continued", lens=_uniform(8, 100, 600, 2), prior=_uniform(8, 1000, 8000, 3)),
        # One 32k prompt: the context of the headline configuration, compute bound.
        dict(L8B, kind="prompt", name="prompt_8b_32k", lens="32768", prior="0"),
        # Four answers to one short fp32 prompt: latency.
        dict(SMALL_F32, kind="shared", name="shared_f32_small", groups="4", shared="1024", own="1,40,17,9"),
        # 32 samples of one 8k prompt half way through 256 generated tokens (the batch-32 decode of the repository).
        dict(L8B, kind="shared", name="shared_8b_8k", groups="32", shared="8192", own=_uniform(32, 1, 256, 4)),
        # Eight prompts of different lengths with one to sixteen answers each; partly filled last pages.
        dict(L8B, kind="shared", name="shared_8b_groups", groups="1,16,8,5,12,2,16,4", shared=_uniform(8, 1000, 32768, 5),
             own=_uniform(64, 1, 1500, 6)),
        # 64 samples over a 128k document at the Llama-3-70B geometry: 512 query rows per kv head, compute begins to count.
        dict(L70B, kind="shared", name="shared_70b_128k", groups="64", shared="131072", own=_uniform(64, 1, 2048, 7)),
        # A few short fp32 prompts come in.
        dict(SMALL_F32, kind="pages", what="admit", name="admit_f32_small", layers=2, lens="1,40,16,17", rows=8, fill=0.5),
        # 16 prompts of up to 4k tokens come in, four layers of keys and values.
        dict(L8B, kind="pages", what="admit", name="admit_8b", layers=4, lens=_uniform(16, 500, 4096, 8), rows=64, fill=0.5),
        # Eight answers to each of eight running prompts: tables, counts and the partly filled last pages of four layers.
        dict(L8B, kind="pages", what="fork", name="fork_8b", layers=4, lens=_uniform(8, 2000, 8192, 9), children=8, share=True),
        # Half of 64 sequences have left: two layers' live pages move together.
        dict(L8B, kind="pages", what="compact", name="compact_8b", layers=2, lens=_uniform(64, 1000, 8192, 10), keep=0.5),
    ]


def _text(values):
    return ",".join(str(x) for x in values)


def _ints(text):
    return [int(x) for x in text.split(",")]


def _uniform(n, lo, hi, seed):
    rng = random.Random(seed)
    return _text(rng.randint(lo, hi) for _ in range(n))


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    hq, hkv, d = rng.choice(DRAWN)
    base = {"dtype": "f32" if rng.random() < 0.25 else "bf16", "q_heads": hq, "kv_heads": hkv, "head_dim": d}
    kind = rng.choice(["prompt", "shared", "pages"])
    while True:
        if kind == "prompt":
            n, hi = _log_uniform(rng, 1, 64), _log_uniform(rng, 8, 32768)
            lens = [_log_uniform(rng, 1, hi) for _ in range(n)]
            far = _log_uniform(rng, 1, 16384) if rng.random() < 0.4 else 0
            prior = [rng.randint(0, far) for _ in lens]
            case = dict(base, kind=kind, lens=_text(lens), prior=_text(prior))
            limit = 2e11 if base["dtype"] == "f32" else 4e12
            if work(case)["flops"] <= limit and sum(lens) + sum(prior) <= 131072:
                return case
        elif kind == "shared":
            groups = [_log_uniform(rng, 1, 64) for _ in range(_log_uniform(rng, 1, 16))]
            hi, own_hi = _log_uniform(rng, 16, 131072), _log_uniform(rng, 1, 4096)
            case = dict(base, kind=kind, groups=_text(groups), shared=_text(_log_uniform(rng, 1, hi) for _ in groups),
                        own=_text(rng.randint(1, own_hi) for _ in range(sum(groups))))
            w = work(case)
            if w["flops"] <= 2e11 and w["bytes"] <= 4e9:
                return case
        else:
            what = rng.choice(["admit", "fork", "compact"])
            n, hi = _log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16384)
            lens = [_log_uniform(rng, 1, hi) for _ in range(n)]
            case = dict(base, kind=kind, what=what, layers=rng.randint(1, 4), lens=_text(lens))
            if what == "admit":
                case.update(rows=n + rng.randint(0, 32), fill=rng.uniform(0.0, 0.8))
            elif what == "fork":
                case.update(children=_log_uniform(rng, 1, 16), share=rng.random() < 0.7)
            else:
                case.update(keep=rng.uniform(0.1, 0.9))
            if sum(lens) * case["layers"] * hkv * d <= 1 << 29 and (what != "fork" or case["children"] * n <= 1024) \
                    and (what != "fork" or case["share"] or sum(lens) * case["children"] <= 131072):
                return case


def work(case):
    """Inputs read once and outputs written once; two operations per multiply-add of the two products."""
    hq, hkv, d, size = case["q_heads"], case["kv_heads"], case["head_dim"], DTYPES[case["dtype"]].itemsize
    if case["kind"] == "prompt":
        lens, prior = _ints(case["lens"]), _ints(case["prior"])
        q, kv = sum(lens), sum(lens) + sum(prior)
        pairs = sum(n * (n + 1) // 2 + n * p for n, p in zip(lens, prior))
        return {"bytes": size * d * (2 * q * hq + 2 * kv * hkv), "flops": 4 * d * hq * pairs}
    if case["kind"] == "shared":
        groups, shared, own_tokens = _ints(case["groups"]), _ints(case["shared"]), sum(_ints(case["own"]))
        tokens = sum(n * s for n, s in zip(groups, shared)) + own_tokens
        return {"bytes": size * d * (2 * sum(groups) * hq + 2 * (sum(shared) + own_tokens) * hkv), "flops": 4 * d * hq * tokens}
    lens = _ints(case["lens"])
    run, pages = 2 * size * d * hkv * case["layers"], [-(-n // PAGE) for n in lens]
    if case["what"] == "admit":
        return {"bytes": 2 * run * sum(lens) + 8 * sum(pages), "flops": 0}
    if case["what"] == "fork":
        copied = sum(n % PAGE if case["share"] else n for n in lens)
        return {"bytes": case["children"] * (2 * run * copied + 8 * sum(pages)), "flops": 0}
    gone, moved = _departed(case), 0
    live = sum(p for p, g in zip(pages, gone) if not g)
    order = _shuffled_pages(case)
    at = 0
    for p, g in zip(pages, gone):
        moved += 0 if g else sum(1 for x in order[at:at + p] if x >= live)
        at += p
    return {"bytes": 2 * run * PAGE * moved + 8 * live, "flops": 0}


def _departed(case):
    lens = _ints(case["lens"])
    rng = random.Random(len(lens) + sum(lens))
    return [rng.random() >= case["keep"] for _ in lens]


def _shuffled_pages(case):
    lens = _ints(case["lens"])
    order = list(range(sum(-(-n // PAGE) for n in lens)))
    random.Random(sum(lens)).shuffle(order)
    return order


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------

def _int32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, shape, dtype, scale=None):
    x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32)
    if scale is not None:
        x *= scale
    return x.to(dtype)


def _key_scale(g, d):
    return torch.exp(0.5 * torch.randn((d,), generator=g, device="cuda"))


def _prompt_inputs(case, seed):
    g, dt, d = _generator(seed), DTYPES[case["dtype"]], case["head_dim"]
    q_lens = _ints(case["lens"])
    kv_lens = [n + p for n, p in zip(q_lens, _ints(case["prior"]))]
    scale = _key_scale(g, d)
    return types.SimpleNamespace(
        case=case, q_lens=q_lens, kv_lens=kv_lens,
        q=_normal(g, (sum(q_lens), case["q_heads"], d), dt),
        k=_normal(g, (sum(kv_lens), case["kv_heads"], d), dt, scale),
        v=_normal(g, (sum(kv_lens), case["kv_heads"], d), dt))


def _shared_inputs(case, seed):
    """A pool in which a group's shared pages appear once; a prefix that ends inside a page has that page copied for every
    member, as a fork leaves it."""
    g, dt, d, hkv = _generator(seed), DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    groups, shared_lens, own_lens = _ints(case["groups"]), _ints(case["shared"]), _ints(case["own"])
    lens, rows, n_pages, at = [], [], 0, 0
    copies = []                                        # (page, page it starts as a copy of, tokens)
    for n, shared in zip(groups, shared_lens):
        full, tail, first_tail = shared // PAGE, shared % PAGE, None
        base = n_pages
        n_pages += full
        for i in range(n):
            length = shared + own_lens[at]
            own_pages = -(-length // PAGE) - full
            rows.append(list(range(base, base + full)) + list(range(n_pages, n_pages + own_pages)))
            if tail:
                if first_tail is None:
                    first_tail = n_pages
                else:
                    copies.append((n_pages, first_tail, tail))
            n_pages += own_pages
            lens.append(length)
            at += 1
    scale = _key_scale(g, d)
    k_pool = _normal(g, (n_pages, hkv, PAGE, d), dt, scale)
    v_pool = _normal(g, (n_pages, hkv, PAGE, d), dt)
    perm = torch.randperm(n_pages, generator=g, device="cuda")
    for page, src, tail in copies:
        for pool in (k_pool, v_pool):
            pool[perm[page], :, :tail] = pool[perm[src], :, :tail]
    table = torch.zeros((len(rows), max(len(r) for r in rows)), dtype=torch.int32, device="cuda")
    for b, r in enumerate(rows):
        table[b, :len(r)] = perm[r[0]:r[0] + len(r)] if r == list(range(r[0], r[0] + len(r))) else perm[torch.tensor(r, device="cuda")]
    return types.SimpleNamespace(
        case=case, groups=groups, shared=shared_lens, lens=lens, k_pool=k_pool, v_pool=v_pool, table=table, seq_lens=_int32(lens),
        shared_lens=_int32(shared_lens), q=_normal(g, (len(lens), case["q_heads"], d), dt))


def _pages_inputs(case, seed):
    g, dt, d, hkv = _generator(seed), DTYPES[case["dtype"]], case["head_dim"], case["kv_heads"]
    lens, what = _ints(case["lens"]), case["what"]
    pages = [-(-n // PAGE) for n in lens]
    s = types.SimpleNamespace(case=case, lens=lens)
    if what == "admit":
        n_rows, max_pages = case["rows"], max(pages)
        n_pages = int(sum(pages) / (1.0 - case["fill"])) + 1
        s.rows = list(range(len(lens)))
    elif what == "fork":
        n_rows, max_pages = len(lens) * (1 + case["children"]), max(pages)
        each = [int(n % PAGE != 0) if case["share"] else p for n, p in zip(lens, pages)]
        n_pages = sum(pages) + case["children"] * sum(each) + 64
        s.parents = [p for p in range(len(lens)) for _ in range(case["children"])]
        s.children = list(range(len(lens), n_rows))
    else:
        n_rows, max_pages, n_pages = len(lens), max(pages), sum(pages)
    scale = _key_scale(g, d)
    s.pools = [(_normal(g, (n_pages, hkv, PAGE, d), dt, scale), _normal(g, (n_pages, hkv, PAGE, d), dt))
               for _ in range(case["layers"])]
    s.table = torch.full((n_rows, max_pages), -1, dtype=torch.int32, device="cuda")
    s.seq_lens = torch.zeros((n_rows,), dtype=torch.int32, device="cuda")
    s.refs = torch.zeros((n_pages,), dtype=torch.int32, device="cuda")
    if what == "admit":
        # other requests hold a random part of the pool (their rows are not in this table)
        taken = torch.randperm(n_pages, generator=g, device="cuda")[:n_pages - sum(pages)]
        s.refs[taken] = 1
        s.starts = _int32([0] + [sum(lens[:i + 1]) for i in range(len(lens))])
        s.new_lens = _int32(lens)
        s.k = [_normal(g, (sum(lens), hkv, d), dt, scale) for _ in range(case["layers"])]
        s.v = [_normal(g, (sum(lens), hkv, d), dt) for _ in range(case["layers"])]
        s.rows_dev = _int32(s.rows)
    else:
        order = _int32(_shuffled_pages(case)) if what == "compact" else torch.randperm(n_pages, generator=g, device="cuda")
        gone, at = (_departed(case) if what == "compact" else [False] * len(lens)), 0
        for b, p in enumerate(pages):
            if not gone[b]:
                s.table[b, :p] = order[at:at + p]
                s.refs[order[at:at + p].long()] = 1
                s.seq_lens[b] = lens[b]
            at += p
        if what == "fork":
            s.parents_dev, s.children_dev = _int32(s.parents), _int32(s.children)
        else:
            s.saved = (s.table.clone(), s.refs.clone())
    return s


def prepare(case, seed):
    if case["kind"] == "prompt":
        s = _prompt_inputs(case, seed)
        if own:
            from interattn_b200 import dense_attention
            s.plan = dense_attention.PromptAttention(s.q_lens, case["q_heads"], case["kv_heads"], case["head_dim"],
                                                     kv_lens=s.kv_lens, dtype=DTYPES[case["dtype"]], device="cuda")
        return s
    if case["kind"] == "shared":
        s = _shared_inputs(case, seed)
        if own:
            from interattn_b200 import dense_attention, ops
            kv = ops.PagedKV(s.k_pool, s.v_pool, s.table, s.seq_lens, s.seq_lens)
            s.plan = dense_attention.SharedPrefixAttention(kv, s.groups, s.shared_lens, case["q_heads"])
        return s
    s = _pages_inputs(case, seed)
    if own:
        from interattn_b200 import page_cache
        s.cache = page_cache.PageCache(s.pools, s.table, s.seq_lens, s.refs)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------

def run(s):
    case = s.case
    if case["kind"] == "prompt":
        return s.plan.run(s.q, s.k, s.v) if own else _plain_prompt(s)
    if case["kind"] == "shared":
        return s.plan.step(s.q) if own else _plain_shared(s)
    if case["what"] == "admit":
        if own:
            s.cache.free(s.rows_dev)
            s.cache.extend(s.rows_dev, s.new_lens)
            for i in range(case["layers"]):
                s.cache.write(i, s.rows_dev, s.starts, s.k[i], s.v[i])
        else:
            _plain_free(s, s.rows)
            _plain_admit(s)
    elif case["what"] == "fork":
        if own:
            s.cache.free(s.children_dev)
            s.cache.fork(s.parents_dev, s.children_dev, share=case["share"])
        else:
            _plain_free(s, s.children)
            _plain_fork(s)
    else:
        # the holes of before are put back first; the moved pages' old places still hold their data
        s.table.copy_(s.saved[0])
        s.refs.copy_(s.saved[1])
        if own:
            s.cache.compact()
        else:
            _plain_compact(s)
    return [s.table, s.seq_lens, s.refs] + [t for pair in s.pools for t in pair]


def _softmax_parts(scores, values):
    """(values weighted by exp(score - max), sum of the weights, max) along the last axis of scores."""
    m = scores.amax(dim=-1, keepdim=True)
    p = torch.exp(scores - m)
    return torch.matmul(p, values), p.sum(dim=-1, keepdim=True), m


def _plain_prompt(s):
    case, out = s.case, torch.empty_like(s.q)
    hkv, d, group = case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]
    at_q = at_k = 0
    for n, m in zip(s.q_lens, s.kv_lens):
        k = s.k[at_k:at_k + m].float().permute(1, 2, 0)                                  # [hkv, d, m]
        v = s.v[at_k:at_k + m].float().transpose(0, 1)                                   # [hkv, m, d]
        q = s.q[at_q:at_q + n].float().view(n, hkv, group, d).permute(1, 2, 0, 3)        # [hkv, group, n, d]
        for lo in range(0, n, 1024):
            hi = min(n, lo + 1024)
            seen = m - n + hi
            scores = torch.matmul(q[:, :, lo:hi].reshape(hkv, group * (hi - lo), d), k[:, :, :seen]) / math.sqrt(d)
            late = torch.arange(seen, device="cuda")[None, :] > torch.arange(m - n + lo, m - n + hi, device="cuda")[:, None]
            scores = scores.view(hkv, group, hi - lo, seen).masked_fill_(late, float("-inf")).view(hkv, -1, seen)
            acc, total, _ = _softmax_parts(scores, v[:, :seen])
            out[at_q + lo:at_q + hi] = (acc / total).view(hkv, group, hi - lo, d).permute(2, 0, 1, 3).reshape(hi - lo, -1, d).to(out.dtype)
        at_q, at_k = at_q + n, at_k + m
    return out


def _plain_shared(s):
    case, out = s.case, torch.empty_like(s.q)
    hkv, d, group = case["kv_heads"], case["head_dim"], case["q_heads"] // case["kv_heads"]

    def tokens(pool, b, lo, hi):
        pages = s.table[b, lo // PAGE:-(-hi // PAGE)].long()
        x = pool[pages].float().transpose(0, 1).reshape(hkv, -1, d)
        return x[:, lo % PAGE:lo % PAGE + hi - lo]

    first = 0
    for n, shared in zip(s.groups, s.shared):
        q = s.q[first:first + n].float().view(n, hkv, group, d).permute(1, 0, 2, 3).reshape(hkv, n * group, d) / math.sqrt(d)
        acc, total, top = _softmax_parts(torch.matmul(q, tokens(s.k_pool, first, 0, shared).transpose(1, 2)),
                                         tokens(s.v_pool, first, 0, shared))
        for i in range(n):
            b, rows = first + i, slice(i * group, (i + 1) * group)
            k, v = tokens(s.k_pool, b, shared, s.lens[b]), tokens(s.v_pool, b, shared, s.lens[b])
            acc1, total1, top1 = _softmax_parts(torch.matmul(q[:, rows], k.transpose(1, 2)), v)
            m = torch.maximum(top[:, rows], top1)
            w0, w1 = torch.exp(top[:, rows] - m), torch.exp(top1 - m)
            o = (acc[:, rows] * w0 + acc1 * w1) / (total[:, rows] * w0 + total1 * w1)
            out[b] = o.reshape(hkv * group, d).to(out.dtype)
        first += n
    return out


def _plain_free(s, rows):
    """Rows give their pages back; what lies past a row's pages in the table stays."""
    index = torch.tensor(rows, device="cuda")
    held = torch.arange(s.table.shape[1], device="cuda")[None, :] < ((s.seq_lens[index] + PAGE - 1) // PAGE)[:, None]
    pages = s.table[index].clamp_min(0).long()
    s.refs.index_put_((pages.view(-1),), -held.view(-1).int(), accumulate=True)
    s.table[index] = torch.where(held, torch.full_like(s.table[index], -1), s.table[index])
    s.seq_lens[index] = 0


def _plain_admit(s):
    lens = s.lens
    free = torch.nonzero(s.refs == 0).view(-1)
    places, at = [], 0
    for b, n in zip(s.rows, lens):
        p = -(-n // PAGE)
        mine = free[at:at + p]
        s.table[b, :p] = mine
        t = torch.arange(n, device="cuda")
        places.append(mine[t // PAGE] * PAGE + t % PAGE)
        at += p
    s.refs[free[:at]] = 1
    s.seq_lens[torch.tensor(s.rows, device="cuda")] = s.new_lens
    place = torch.cat(places)
    for (k_pool, v_pool), k, v in zip(s.pools, s.k, s.v):
        k_pool[place // PAGE, :, place % PAGE] = k
        v_pool[place // PAGE, :, place % PAGE] = v


def _plain_fork(s):
    case, free, at = s.case, torch.nonzero(s.refs == 0).view(-1), 0
    src, dst = [], []
    for parent, child in zip(s.parents, s.children):
        n = s.lens[parent]
        pages, kept = -(-n // PAGE), (n // PAGE if case["share"] else 0)
        s.table[child, :kept] = s.table[parent, :kept]
        s.refs[s.table[parent, :kept].long()] += 1
        new = free[at:at + pages - kept]
        s.table[child, kept:pages] = new
        src.append(s.table[parent, kept:pages].long())
        dst.append(new)
        s.seq_lens[child] = n
        at += pages - kept
    s.refs[free[:at]] = 1
    src, dst = torch.cat(src), torch.cat(dst)
    for pair in s.pools:
        for pool in pair:
            pool[dst] = pool[src]


def _plain_compact(s):
    live = s.refs > 0
    n_live = live.sum()
    index = torch.arange(live.numel(), device="cuda")
    src, dst = torch.nonzero(live & (index >= n_live)).view(-1), torch.nonzero(~live & (index < n_live)).view(-1)
    for pair in s.pools:
        for pool in pair:
            pool[dst] = pool[src]
    s.refs[dst] = s.refs[src]
    s.refs[src] = 0
    index[src] = dst
    held = torch.arange(s.table.shape[1], device="cuda")[None, :] < ((s.seq_lens + PAGE - 1) // PAGE)[:, None]
    s.table.copy_(torch.where(held, index[s.table.clamp_min(0).long()].int(), s.table))


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------

def exact(case, seed):
    """Row by row from the definition, in float64; pages are moved and counted, not computed."""
    if case["kind"] == "pages":
        return None
    d, group = case["head_dim"], case["q_heads"] // case["kv_heads"]
    if case["kind"] == "prompt":
        s = _prompt_inputs(case, seed)
        out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for n, m in zip(s.q_lens, s.kv_lens):
            for h in range(case["q_heads"]):
                keys, values = s.k[k0:k0 + m, h // group].double(), s.v[k0:k0 + m, h // group].double()
                for lo in range(0, n, 4096):
                    hi = min(n, lo + 4096)
                    logits = s.q[q0 + lo:q0 + hi, h].double() @ keys.T * d ** -0.5
                    visible = torch.ones((hi - lo, m), dtype=torch.bool, device="cuda").tril_(m - n + lo)
                    out[q0 + lo:q0 + hi, h] = torch.softmax(logits.masked_fill_(~visible, -math.inf), dim=-1) @ values
            q0, k0 = q0 + n, k0 + m
        return out
    s = _shared_inputs(case, seed)
    out = torch.zeros(s.q.shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s.lens):
        pages = s.table[b, :-(-length // PAGE)].long()
        for kv in range(case["kv_heads"]):
            keys, values = (pool[pages, kv].double().reshape(-1, d)[:length] for pool in (s.k_pool, s.v_pool))
            heads = slice(kv * group, (kv + 1) * group)
            out[b, heads] = torch.softmax(s.q[b, heads].double() @ keys.T * d ** -0.5, dim=-1) @ values
    return out
