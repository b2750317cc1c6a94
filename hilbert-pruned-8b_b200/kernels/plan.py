"""Launch-shape decisions of the host that need no device: pure functions, tested on the CPU."""
from __future__ import annotations


def decode_splits(sequences: int, kv_heads: int, max_pages: int, cta_slots: int) -> int:
    """Key splits of split-K decode attention for ``sequences`` x ``kv_heads`` (sequence, kv head)
    pairs whose longest cache holds ``max_pages`` pages, on a device that holds ``cta_slots``
    of the kernel's CTAs at once.

    At most 16 splits and at most one for every eight pages (measured: more splits cost more in
    the combination than they gain).  One wave of the resident CTAs if that fills the device:
    batch 8 at 8192 tokens takes 4 splits on 296 slots.  Where one wave would leave a third of
    the device idle (batch 24: 192 CTAs) or a second wave would (batch 48: 384 CTAs), the
    splits that fill whole waves best, of 32 pages or more each (12 % of a step at batch 48)."""
    slots = max(1, cta_slots)
    pairs = max(1, sequences * kv_heads)
    limit = max(1, min(16, -(-max_pages // 8)))

    def fill(s: int) -> float:            # share of the waves' CTA slots that have work
        ctas = pairs * s
        return ctas / (-(-ctas // slots) * slots)

    best = max(1, min(slots // pairs, limit))
    if fill(best) < 0.8:
        for s in range(1, limit + 1):
            if -(-max_pages // s) >= 32 and fill(s) - 0.01 * s > fill(best) - 0.01 * best + 0.1:
                best = s
    return best


def few_groups(new, lengths, heads: int, limit: int):
    """Which sequences of a step of few tokens run at once: ``[(first sequence, their number, first token, their number, rows of the longest)]``,
    neighbours, in order.  The scores of a group (``heads`` times its tokens times its longest sequence's rows, in whole pages) are at most
    ``limit`` floats, or those of one sequence's tokens: one long sequence among many short ones would else cost every token a row of its
    length (64 single tokens, one of them behind 131072 rows, 32 heads: 1 GB).  A sequence without new tokens goes with one that has some."""
    parts, first, longest = [], 0, 1                              # [first sequence, their number, their tokens, rows of the longest]
    for b, (n, ln) in enumerate(zip(new, lengths)):
        longest = max(longest, ln)
        if n > 0:
            parts.append([first, b + 1 - first, n, longest])
            first, longest = b + 1, 1
    if parts:
        parts[-1][1] += len(new) - first
        parts[-1][3] = max(parts[-1][3], longest)
    groups, at = [], 0
    for b, count, n, ln in parts:
        if groups and heads * (groups[-1][3] + n) * (-(-max(groups[-1][4], ln) // 64) * 64) <= limit:
            b0, seqs, t0, tokens, rows = groups[-1]
            groups[-1] = (b0, seqs + count, t0, tokens + n, max(rows, ln))
        else:
            groups.append((b, count, at, n, ln))
        at += n
    return groups


def few_splits(pages, kv_heads: int, cta_slots: int):
    """Shares of a sequence's pages in a step of few tokens that keeps its scores: (the most of a sequence, the fewest pages of one);
    ``pages``: how many each block of tokens sees.  As ``decode_splits``, but down to a page each (64 shares at most) while the device has room, since
    a second kernel follows in any case.  With blocks of unequal lengths shares of about equal size that take one round of the device (32 of a
    sequence at most)."""
    blocks, most, total = max(1, len(pages)), max(pages, default=1), sum(pages)
    if 4 * most * blocks <= 5 * total or total == 0:
        room = max(1, cta_slots) // (blocks * kv_heads)
        return max(1, min(max(decode_splits(blocks, kv_heads, most, cta_slots), min(most, 64, room)), most)), 1
    size = max(1, -(-total * kv_heads // cta_slots), -(-most // 32))
    while size < most and kv_heads * sum(-(-n // size) for n in pages) > cta_slots:
        size += 1
    return -(-most // size), size


def chunk_shares(new, lengths, window: int, span: int, keys: int, units: int, row_floats: int, slots: int, own: float, join: float):
    """How the keys of blocks of queries are shared out over blocks of threads: (the most shares of one block of queries, the most tiles of
    ``keys`` keys in a share, the new tokens of sequences that may be cut).  ``new`` tokens and ``lengths`` of the sequences, blocks of ``span`` tokens, ``units`` heads or pairs of heads,
    ``row_floats`` floats that a share leaves per token, on a device with ``slots`` places.

    A sequence's blocks start with the ones that see the most keys (sequences as the kernels take them: from the step's last to its
    first, whatever they see), so a step lasts about as long as its work divided by the places, or as its longest block.  Where that is the longer of the two, blocks are cut: with shares of at most t tiles a step lasts about the lesser of
    (work / places + t) and t times the rounds that its shares need.  To start and end a share takes the time of ``own``
    tiles, the kernel that joins the shares that of ``join``.  (Measured: the tensor-core kernel 7 to 9 us against 1.6 to 2 us for a tile of 128
    keys, the kernel for every type about 3 us like its tile of 64.)  The partial results are at most 256 MB in all."""
    blocks = []                                                            # per sequence: blocks, tiles that one may see, new tokens
    work = 0.0
    for n, ln in zip(new, lengths):
        if n > 0:
            nb = -(-n // span)
            most = -(-min(ln, window + span if window else ln) // keys) + (1 if window else 0)
            least = min(most, -(-(ln - n + 1) // keys))
            blocks.append((nb * units, most, n))
            work += nb * units * (most + least) / 2
    if not blocks:
        return 1, 1, 0
    longest = max(t for _, t, _ in blocks)
    count = sum(c for c, _, _ in blocks)
    ideal = (work + own * count) / slots
    if longest <= 4 or longest + own <= 1.25 * ideal:
        return 1, longest, 0
    best, shares, tiles = max(longest + own, min(ideal + longest / 2, (longest + own) * -(-count // slots))), 1, longest
    for s in (2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32):
        t = -(-longest // s)
        if s > longest or s * row_floats * sum(new) > 64 << 20:
            break
        count = sum(c * -(-m // t) for c, m, _ in blocks)
        cost = min((work + own * count) / slots + t, (t + own) * -(-count // slots)) + join
        if cost < best:
            best, shares, tiles = cost, s, t
    return shares, tiles, sum(n for _, m, n in blocks if m > tiles)


def mass_splits(new, lengths, window: int, tile: int, span: int, kv_heads: int, group: int, cta_slots: int) -> int:
    """Shares of the weights' kernel, whose block takes a tile of keys and goes through the tiles of ``span`` queries of each head that see
    it.  Under a causal mask the first keys are seen by every query and the last by few, and a sequence's heaviest tiles start first: shares
    so that a heaviest one is about an even share of the work (4096-token prompt: 2, 242 us in all, against 323 with 1 and 255 with 5)."""
    most = total = 0
    for n, ln in zip(new, lengths):
        if n > 0:
            blocks = -(-n // span)
            seen = min(blocks, (window + tile) // span + 1) if window else blocks
            most = max(most, seen)
            old, fresh = (ln - n) // tile, n // tile + 1                  # tiles of older rows, of the step's own
            if window:
                old = min(old, -(-window // tile))
            total += old * seen + fresh * (seen + 1) / 2 if not window else (old + fresh) * (seen + 1) / 2
    if not most:
        return 1
    even = max(1.0, total * group * kv_heads / max(1, cta_slots))
    return max(1, min(16, most * group, round(most * group / even)))


def select_shape(lists: int, rows: int, sms: int):
    """(threads, blocks in a cluster) for choosing among ``rows`` rows in each of ``lists`` lists.  A thread keeps up to 32 rows in
    registers: 512 threads (two blocks to an SM) where that holds a list, else 1024 and a cluster that does.  With few lists, more
    blocks to a list while the device has SMs without one and a thread would still have 8 rows or more."""
    per_thread = 32
    threads = 512 if rows <= 512 * per_thread and lists > sms // 2 else 1024
    cluster = 1
    while cluster < 8 and rows > cluster * threads * per_thread:
        cluster *= 2
    while cluster < 8 and 2 * cluster * lists <= sms and rows >= 2 * cluster * threads * 8:
        cluster *= 2
    return threads, cluster
