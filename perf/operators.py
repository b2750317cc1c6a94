"""What the operators of a bounded cache are measured on: attention that adds up every cached row's weight (chunks of new
tokens and single tokens), the choice of the rows that stay, and their move to the front of the pages.

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, with ``own`` true, by the
library's kernels; ``exact`` gives the same outputs from the definitions in 64 bits.

The cache is paged as the library's is: ``[entries,] pages, kv_heads, 64, head size``, pages in any order, rows behind a
sequence's end holding other values.  Mass is ``[entries,] pages, kv_heads, 64`` in float32.
"""
import math
from types import SimpleNamespace

import torch

own = False

PAGE = 64
_TYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # a chunk of a prompt that starts a conversation, a layer of the 8B sizes
        _chunk("chunk_prompt", 32, 8, 128, "0", "4096", 0, True, "bfloat16"),
        # a chunk of a long prompt behind 30000 rows, a layer of the 8B sizes
        _chunk("chunk_long_past", 32, 8, 128, "30001", "2048", 0, False, "bfloat16"),
        # prompts and conversations of unequal lengths in one step, a layer of the 1B sizes
        _chunk("chunk_ragged", 32, 8, 64, "0,517,64,1999,3,0,4100", "700,33,129,1,511,64,257", 0, False, "bfloat16"),
        # drafted tokens of several conversations checked in one step
        _chunk("chunk_few", 32, 8, 128, "2047,8000,515,4096", "5,5,3,4", 0, False, "bfloat16"),
        # the true 32-bit path with a head size and a group of no power of two, a window
        _chunk("chunk_f32_odd", 6, 2, 80, "0,333", "190,75", 200, False, "float32"),
        # one short conversation: where latency counts
        _chunk("token_small", 32, 8, 64, "299", "1", 0, False, "bfloat16"),
        # a batch of conversations, one token each, a layer of the 8B sizes
        _chunk("token_batch", 32, 8, 128, "8191,8000,7000,8191,6001,8190,8192,4444", "1,1,1,1,1,1,1,1", 0, False, "bfloat16"),
        # two long documents
        _chunk("token_long", 32, 8, 128, "100000,65537", "1,1", 0, False, "bfloat16"),
        # one layer's choice for short conversations, one of them below its budget
        _select("select_small", 1, 8, "700,100,257", 128, 4, 32),
        # all layers of the 8B sizes at once, a long prompt cut to an eighth
        _select("select_layers", 32, 8, "16384", 2048, 4, 256),
        # one layer's rows moved into pages of their own, the 32-bit cache
        _rows("rows_small", 1, 2, 80, "700,257", 128, 4, 32, "float32"),
        # all layers of the 8B sizes at once
        _rows("rows_layers", 32, 8, 128, "16384", 2048, 4, 256, "bfloat16"),
    ]


def _chunk(name, heads, kv_heads, head_dim, past, new, window, first_weights, dtype):
    """``first_weights``: the mass starts with this step (no earlier sum is added)."""
    return {"name": name, "kind": "attention", "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "past": past, "new": new,
            "window": window, "first_weights": first_weights, "dtype": dtype}


def _select(name, entries, kv_heads, lengths, budget, first, recent):
    return {"name": name, "kind": "select", "entries": entries, "kv_heads": kv_heads, "lengths": lengths, "budget": budget, "first": first,
            "recent": recent}


def _rows(name, entries, kv_heads, head_dim, lengths, budget, first, recent, dtype):
    return {"name": name, "kind": "rows", "entries": entries, "kv_heads": kv_heads, "head_dim": head_dim, "lengths": lengths,
            "budget": budget, "first": first, "recent": recent, "dtype": dtype}


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["chunk", "chunk", "few", "token", "token", "select", "rows"])
    if kind in ("chunk", "few", "token"):
        kv = rng.choice([1, 2, 4, 8])
        group = rng.choice([1, 2, 3, 4, 8])
        while kv * group > 32:
            group = rng.choice([1, 2, 4])
        dtype = "bfloat16" if rng.random() < 0.75 else "float32"
        hd = rng.choice([64, 128, 128]) if dtype == "bfloat16" and rng.random() < 0.8 else 8 * rng.randint(3, 24)
        plain = dtype == "float32" or hd not in (64, 128)
        window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
        n = rng.randint(1, 8)
        if kind == "token":
            longest = _log_int(rng, 64, 16384 if plain else 65536)
            past = [rng.randint(longest // 2, longest) for _ in range(n)]
            new = [1] * n
        elif kind == "few":
            longest = _log_int(rng, 64, 4096 if plain else 16384)
            past = [rng.randint(0, longest) for _ in range(n)]
            new = [rng.randint(1, 8) for _ in range(n)]
        else:
            n = rng.randint(1, 5)
            past = [0 if rng.random() < 0.3 else _log_int(rng, 1, 700 if plain else 8000) for _ in range(n)]
            new = [_log_int(rng, 1, 400 if plain else 2000) for _ in range(n)]
        return {k: v for k, v in _chunk("", kv * group, kv, hd, ",".join(map(str, past)), ",".join(map(str, new)), window,
                                        rng.random() < 0.3, dtype).items() if k != "name"}
    entries, kv, n = rng.choice([1, 2, 8, 16, 28]), rng.choice([1, 2, 4, 8]), rng.randint(1, 4)
    longest = _log_int(rng, 100, 131072 // 8 if entries > 2 else 131072)
    if kind == "rows" or n > 1:
        longest = min(longest, 16384)
    if entries * kv * n > 256:
        n = 1
    budget = min(_log_int(rng, 48, 4096), 2048 if entries * kv * n > 64 else 4096)
    first, recent = rng.choice([0, 1, 4, 16]), rng.randint(0, 32)
    lengths = ",".join(str(rng.randint(max(1, longest // 3), longest)) for _ in range(n))
    if kind == "select":
        case = _select("", entries, kv, lengths, budget, first, recent)
    else:
        hd = rng.choice([64, 80, 128, 128])
        case = _rows("", entries, kv, hd, lengths, budget, first, recent, rng.choice(["bfloat16", "bfloat16", "float32"]))
    return {k: v for k, v in case.items() if k != "name"}


# ----------------------------------------------------------------------------------------------------------- inputs
def _ints(text):
    return [int(x) for x in text.split(",")]


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _tables(lengths, gen, extra, width=None):
    """Pages in any order for rows of each length (-1 where a sequence has none), and how many pages the cache has."""
    counts = [_pages(n) for n in lengths]
    total = sum(counts) + extra
    order = torch.randperm(total, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), width or max(1, max(counts))), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at: at + c]
        at += c
    return table, total, order[at:]


def _mass_values(shape, gen):
    """Sums of softmax weights as they build up: a few rows hold most of it, many hold very little, and many are alike."""
    m = torch.empty(shape, dtype=torch.float32, device="cuda").uniform_(-9.0, 1.0, generator=gen).exp_()
    return torch.where(m < 0.002, (m * 4096).round() / 4096, m)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["kind"] == "attention":
        return _prepare_attention(case, gen)
    lengths = _ints(case["lengths"])
    s = SimpleNamespace(case=case, kind=case["kind"], lengths=lengths, first=case["first"], recent=case["recent"], budget=case["budget"])
    E, kv, B = case["entries"], case["kv_heads"], len(lengths)
    spare = B * _pages(case["budget"]) if case["kind"] == "rows" else 0
    s.table, total, rest = _tables(lengths, gen, spare + 3)
    s.lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s.mass = _mass_values((E, total, kv, PAGE), gen)
    s.kept = torch.empty(E, B, kv, case["budget"], dtype=torch.int32, device="cuda")
    if case["kind"] == "rows":
        dt, hd = _TYPES[case["dtype"]], case["head_dim"]
        s.k = torch.empty(E, total, kv, PAGE, hd, dtype=dt, device="cuda").normal_(generator=gen)
        s.v = torch.empty(E, total, kv, PAGE, hd, dtype=dt, device="cuda").normal_(generator=gen)
        s.to = rest[:spare].view(B, _pages(case["budget"])).contiguous()
        s.kept.copy_(_chosen(s))
    return s


def _prepare_attention(case, gen):
    past, new = _ints(case["past"]), _ints(case["new"])
    lengths = [p + n for p, n in zip(past, new)]
    heads, kv, hd, dt = case["heads"], case["kv_heads"], case["head_dim"], _TYPES[case["dtype"]]
    T, B = sum(new), len(new)
    table, total, _ = _tables(lengths, gen, 3)
    s = SimpleNamespace(case=case, kind="attention", past=past, new=new, lengths=lengths, heads=heads, kv=kv, hd=hd, window=case["window"] or None,
                        scale=1.0 / math.sqrt(hd))
    # queries as they lie in a step: the first columns of the projections' rows
    s.qkv = torch.empty(T, (heads + 2 * kv) * hd, dtype=dt, device="cuda").normal_(generator=gen)
    s.k = torch.empty(total, kv, PAGE, hd, dtype=dt, device="cuda").normal_(generator=gen)
    s.v = torch.empty(total, kv, PAGE, hd, dtype=dt, device="cuda").normal_(generator=gen)
    # a few rows that many queries look at
    s.k[:, :, 5].mul_(1.5)
    s.before = None if case["first_weights"] else _mass_values((total, kv, PAGE), gen)
    s.mass = torch.zeros(total, kv, PAGE, dtype=torch.float32, device="cuda")
    s.out = torch.zeros(T, heads * hd, dtype=dt, device="cuda")
    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s.step = SimpleNamespace(
        num_tokens=T, num_seqs=B, page_tables=[table], positions=ints([p + i for p, n in zip(past, new) for i in range(n)]),
        tok_seq=ints([b for b, n in enumerate(new) for _ in range(n)]), seq_start=ints(starts), seq_pos0=ints(past), seq_len=ints(lengths),
        max_new=max(new), max_len=max(lengths), is_decode=all(n == 1 for n in new), host_new=new, host_len=lengths, shared={}, tag="")
    s.cache = SimpleNamespace(k=s.k, v=s.v, group=0, window=s.window)
    s.table = table
    return s


# ------------------------------------------------------------------------------------------------------ plain forms
_ops = None


def _library():
    global _ops
    if _ops is None:
        from hilbert_pruned_8b_b200.kernels.ops import Ops
        _ops = Ops("cuda:0")
    return _ops


def run(s):
    if s.kind == "attention":
        if own:
            _library().attention_mass(s.qkv, s.heads, s.kv, s.hd, s.cache, s.step, s.out, s.scale, s.window, s.mass, before=s.before)
            return s.out, s.mass
        return _attention(s)
    if s.kind == "select":
        if own:
            _library().evict_select(s.mass, s.table, s.lens, s.first, s.recent, s.kept)
            return s.kept
        return _chosen(s)
    if own:
        _library().evict_rows(s.kept, s.k, s.v, s.mass, s.table, to_table=s.to)
        return s.k, s.v, s.mass
    return _moved(s)


def _attention(s):
    """All sequences at once, padded to the longest."""
    st, G = s.step, s.heads // s.kv
    B, n, W = st.num_seqs, st.max_new, s.table.shape[1]
    L = W * PAGE
    row = (st.positions - st.seq_pos0[st.tok_seq]).long()
    q = torch.zeros(B, n, s.heads * s.hd, device="cuda")
    q[st.tok_seq.long(), row] = s.qkv[:, : s.heads * s.hd].float()
    q = q.view(B, n, s.kv, G, s.hd).permute(0, 2, 3, 1, 4).reshape(B, s.kv, G * n, s.hd)
    pages = s.table.clamp(min=0).long()
    k = s.k[pages].float().permute(0, 2, 1, 3, 4).reshape(B, s.kv, L, s.hd)
    v = s.v[pages].float().permute(0, 2, 1, 3, 4).reshape(B, s.kv, L, s.hd)
    key = torch.arange(L, device="cuda")
    pos = st.seq_pos0[:, None] + torch.arange(n, device="cuda")[None]                        # [B, n]
    there = pos < st.seq_len[:, None]
    seen = (key[None, None] <= pos[:, :, None]) & there[:, :, None]
    if s.window:
        seen &= key[None, None] > pos[:, :, None] - s.window
    v = v * (key[None] < st.seq_len[:, None])[:, None, :, None]                           # rows behind the end count for nothing
    w = torch.matmul(q, k.transpose(2, 3)).mul_(s.scale).view(B, s.kv, G, n, L)
    w.masked_fill_(~seen[:, None, None], float("-inf"))
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == float("-inf"), torch.zeros_like(top), top)).exp_()
    w.div_(w.sum(-1, keepdim=True).clamp(min=1e-37))
    o = torch.matmul(w.view(B, s.kv, G * n, L), v).view(B, s.kv, G, n, s.hd).permute(0, 3, 1, 2, 4).reshape(B, n, -1)
    out = o[st.tok_seq.long(), row].to(s.out.dtype)
    m = w.sum((2, 3))                                                                     # [B, kv, L]
    if s.before is not None:
        old = s.before[pages].permute(0, 2, 1, 3).reshape(B, s.kv, L)
        m = m + old * (key[None] < st.seq_pos0[:, None])[:, None]
    b, j = torch.nonzero(key[None] < st.seq_len[:, None], as_tuple=True)
    mass = torch.zeros_like(s.mass)
    mass[pages[b, j // PAGE], :, j % PAGE] = m[b, :, j]
    return out, mass


def _chosen(s):
    E, kv, B = s.mass.shape[0], s.mass.shape[2], len(s.lengths)
    pages = s.table.clamp(min=0).long()
    L = s.table.shape[1] * PAGE
    m = s.mass[:, pages].permute(0, 1, 3, 2, 4).reshape(E, B, kv, L)
    key, ln = torch.arange(L, device="cuda"), s.lens.long()[None, :, None, None]
    always = (key < s.first) | (key >= ln - s.recent) | (ln <= s.budget)
    m = torch.where(always, torch.full_like(m, float("inf")), m).masked_fill_(key >= ln, float("-inf"))
    order = torch.sort(m, dim=-1, descending=True, stable=True).indices                       # ties: the lower row first
    n = min(s.budget, L)
    top = order[..., :n]
    top = torch.where(torch.arange(n, device="cuda") < ln, top, torch.full_like(top, L))     # fewer rows than the budget
    top = torch.sort(top, dim=-1).values
    kept = torch.full((E, B, kv, s.budget), -1, dtype=torch.int32, device="cuda")
    kept[..., :n] = torch.where(top < L, top, torch.full_like(top, -1)).to(torch.int32)
    return kept


def _moved(s):
    """The kept rows in the pages of ``to``; everything else as it was."""
    e, b, h, j = torch.nonzero(s.kept >= 0, as_tuple=True)
    src = s.kept[e, b, h, j].long()
    sp, dp = s.table[b, src // PAGE].long(), s.to[b, j // PAGE].long()
    for x in (s.k, s.v, s.mass):
        x[e, dp, h, j % PAGE] = x[e, sp, h, src % PAGE]
    return s.k, s.v, s.mass


# ------------------------------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if s.kind == "rows":
        return _exact_rows(s)
    if s.kind == "select":
        return None                                   # whole numbers: the plain form's have to be met
    G = s.heads // s.kv
    out = torch.zeros(s.out.shape, dtype=torch.float64, device="cuda")
    mass = torch.zeros(s.mass.shape, dtype=torch.float64, device="cuda")
    t0 = 0
    for b, (p0, n) in enumerate(zip(s.past, s.new)):
        ln = p0 + n
        j = torch.arange(ln, device="cuda")
        page = s.table[b].long()[j // PAGE]
        i = torch.arange(p0, ln, device="cuda")
        hidden = j[None] > i[:, None]
        if s.window:
            hidden |= j[None] <= i[:, None] - s.window
        for g in range(s.kv):
            k, v = s.k[page, g, j % PAGE].double(), s.v[page, g, j % PAGE].double()
            total = torch.zeros(ln, dtype=torch.float64, device="cuda")
            for h in range(g * G, (g + 1) * G):
                q = s.qkv[t0: t0 + n, h * s.hd: (h + 1) * s.hd].double()
                w = torch.softmax((q @ k.T * s.scale).masked_fill(hidden, float("-inf")), dim=-1)
                out[t0: t0 + n, h * s.hd: (h + 1) * s.hd] = w @ v
                total += w.sum(0)
            if s.before is not None:
                total[:p0] += s.before[page[:p0], g, j[:p0] % PAGE].double()
            mass[page, g, j % PAGE] = total
        t0 += n
    return out, mass


def _exact_rows(s):
    k, v, mass = s.k.clone(), s.v.clone(), s.mass.clone()
    kept, table, to = s.kept.cpu(), s.table.cpu(), s.to.cpu()
    for e in range(kept.shape[0]):
        for b in range(kept.shape[1]):
            for h in range(kept.shape[2]):
                src = kept[e, b, h][kept[e, b, h] >= 0].long()
                j = torch.arange(len(src))
                sp, dp = table[b].long()[src // PAGE].cuda(), to[b].long()[j // PAGE].cuda()
                so, do = (src % PAGE).cuda(), (j % PAGE).cuda()
                for x, y in ((s.k, k), (s.v, v), (s.mass, mass)):
                    y[e, dp, h, do] = x[e, sp, h, so]
    return k.double(), v.double(), mass.double()


# ------------------------------------------------------------------------------------------------------------ work
def work(case):
    """Every input read once, every output written once; of the cache the rows that some query of the step sees."""
    kv = case["kv_heads"]
    if case["kind"] == "attention":
        es, hd, H = (2 if case["dtype"] == "bfloat16" else 4), case["head_dim"], case["heads"]
        pairs = rows = 0
        for p0, n in zip(_ints(case["past"]), _ints(case["new"])):
            w = case["window"] or p0 + n
            rows += p0 + n - max(0, p0 - w + 1)
            # the token at position p sees min(p + 1, w) rows
            short = max(0, min(p0 + n, w) - p0)
            pairs += short * (2 * p0 + short + 1) // 2 + (n - short) * w
        T = sum(_ints(case["new"]))
        mass = rows * kv * 4 * (1 if case["first_weights"] else 2)
        return {"bytes": 2 * T * H * hd * es + 2 * rows * kv * hd * es + mass, "flops": 4 * hd * H * pairs}
    lengths = _ints(case["lengths"])
    E, budget = case["entries"], case["budget"]
    if case["kind"] == "select":
        return {"bytes": 4 * E * kv * (sum(lengths) + len(lengths) * budget), "flops": E * kv * sum(lengths)}
    es = 2 if case["dtype"] == "bfloat16" else 4
    kept = sum(min(n, budget) for n in lengths)
    return {"bytes": E * kv * kept * (2 * (2 * case["head_dim"] * es + 4) + 4), "flops": 0}
