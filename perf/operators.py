"""The serving operators around the compressed cache, as measured cases.

Three operators that a step of speculative decoding runs one after another:

* ``tree``: attention of a tree of drafted tokens over the paged compressed
  cache (a tree of one node is the single-token form);
* ``pages``: forking sequences, compacting the cached rows that a step keeps,
  copying rows out, freeing;
* ``sample``: temperature, top-k, top-p and min-p sampling from given uniform
  random numbers.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
through the package's entry points.
"""

import math
import random

import torch

own = False

D = 64
PAGE = 256
# Centroids of the cache's Gaussian codebooks by their bits, in 1/32768
# (the on-device format's integers).
CENTROIDS = {
    2: (-49490, -14835, 14835, 49490),
    3: (-70498, -44018, -24759, -8027, 8027, 24759, 44018, 70498),
    4: (-89465, -67707, -52923, -41069, -30794, -21451, -12667, -4189,
        4189, 12667, 21451, 30794, 41069, 52923, 67707, 89465),
}


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------

def listed():
    return [
        # one token of one short conversation: nothing but latency
        dict(name="tree token, 100 rows", op="tree", batch=1, context=99, nodes=1, kv_heads=8, groups=4,
             key_bits=4, value_bits=2, ragged=False),
        # a chat batch verifying small trees, each at its own length
        dict(name="tree 8 nodes, 16 seqs", op="tree", batch=16, context=16000, nodes=8, kv_heads=8, groups=4,
             key_bits=4, value_bits=2, ragged=True),
        # one long document, a wide tree
        dict(name="tree 64 nodes, 32K", op="tree", batch=1, context=32768, nodes=64, kv_heads=8, groups=4,
             key_bits=4, value_bits=2, ragged=False),
        # the 3-bit variant, an odd tree, odd lengths
        dict(name="tree 27 nodes, 3b/3b", op="tree", batch=6, context=9001, nodes=27, kv_heads=8, groups=4,
             key_bits=3, value_bits=3, ragged=True),
        # one token over the longest single-GPU context: bound by the cache's bytes
        dict(name="tree token, 1M", op="tree", batch=1, context=1048575, nodes=1, kv_heads=8, groups=4,
             key_bits=4, value_bits=2, ragged=False),
        # a full batch of wide trees: bound by the matrix products and exponentials
        dict(name="tree 64 nodes, 16 seqs", op="tree", batch=16, context=32768, nodes=64, kv_heads=8, groups=4,
             key_bits=4, value_bits=2, ragged=False),
        # one sequence forked, the accepted path of its tree kept
        dict(name="pages path of 5 of 64", op="pages", kind="accept", batch=1, context=1000, nodes=64, keep=5,
             kv_heads=8, key_bits=4, value_bits=2),
        # the same for a batch, at odd lengths
        dict(name="pages path, 32 seqs", op="pages", kind="accept", batch=32, context=2047, nodes=48, keep=7,
             kv_heads=8, key_bits=3, value_bits=3),
        # history eviction: half of a long sequence's rows are kept and moved together
        dict(name="pages evict half of 128K", op="pages", kind="evict", batch=1, context=131072, nodes=0,
             keep=65536, kv_heads=8, key_bits=4, value_bits=2),
        # the next token of one sequence
        dict(name="sample 1 x 32000", op="sample", rows=1, vocab=32000, dtype="float32", pad=0, filters="kp"),
        # every node of a batch's trees, each row with its own settings
        dict(name="sample 256 x 128000", op="sample", rows=256, vocab=128000, dtype="bfloat16", pad=0,
             filters="mixed"),
        # unfiltered sampling reads all logits and all random numbers; rows of a wider buffer
        dict(name="sample 100 x 50003", op="sample", rows=100, vocab=50003, dtype="float32", pad=61,
             filters="none"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("tree", "tree", "pages", "sample"))
    if op == "tree":
        batch, nodes = _log_int(rng, 1, 32), _log_int(rng, 1, 64)
        kv_heads, groups = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8))
        key_bits, value_bits = rng.choice(((4, 2), (4, 2), (3, 3)))
        # at most the largest listed case's products, and a 1M cache's rows
        most = min(16 * 64 * 32 * 32768 // (batch * nodes * kv_heads * groups), 8 * 1048575 // (batch * kv_heads),
                   1048575)
        return dict(op="tree", batch=batch, context=_log_int(rng, 1, most), nodes=nodes, kv_heads=kv_heads,
                    groups=groups, key_bits=key_bits, value_bits=value_bits, ragged=rng.random() < 0.7)
    if op == "pages":
        key_bits, value_bits = rng.choice(((4, 2), (3, 3)))
        kv_heads = rng.choice((1, 2, 4, 8))
        if rng.random() < 0.6:
            nodes = _log_int(rng, 2, 64)
            return dict(op="pages", kind="accept", batch=_log_int(rng, 1, 32), context=_log_int(rng, 1, 16384),
                        nodes=nodes, keep=rng.randint(1, nodes), kv_heads=kv_heads, key_bits=key_bits,
                        value_bits=value_bits)
        context = _log_int(rng, 2, 131072)
        return dict(op="pages", kind="evict", batch=1, context=context, nodes=0, keep=rng.randint(1, context // 2),
                    kv_heads=kv_heads, key_bits=key_bits, value_bits=value_bits)
    return dict(op="sample", rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 300, 128000),
                dtype=rng.choice(("float32", "bfloat16", "float16")), pad=rng.choice((0, 0, 1, 8, 61)),
                filters=rng.choice(("none", "k", "p", "m", "kp", "kpm", "mixed", "mixed")))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _contexts(case):
    """Cached tokens before the drafted ones, for each sequence."""
    b, t = case["batch"], case["context"]
    if not case.get("ragged"):
        return [t] * b
    return [max(1, t * (i + 1) // b - i % 5) for i in range(b)]


def _parents(case):
    """A drafted tree for each sequence: node i's parent comes before it, -1 is the context's last token."""
    rng = random.Random(1000 * case["batch"] + case["nodes"])
    out = []
    for _ in range(case["batch"]):
        out.append([-1 if i == 0 or rng.random() < 0.1 else rng.randint(max(0, i - 12), i - 1)
                    for i in range(case["nodes"])])
    return out


def _kept(case, seed):
    """(batch, keep) on the host: the offsets of the rows that stay, rising,
    after a sequence's first `context` rows (accept) or from its first row (evict)."""
    among = case["nodes"] if case["kind"] == "accept" else case["context"]
    g = torch.Generator().manual_seed(seed)
    return torch.rand((case["batch"], among), generator=g).argsort(1)[:, :case["keep"]].sort(1).values


def _pack(codes, bits):
    """Codes (..., 64) -> bytes (..., 8 * bits), least significant bits first."""
    c = codes.reshape(*codes.shape[:-1], 8, 8).to(torch.int64)
    word = (c << (bits * torch.arange(8, device=c.device))).sum(-1)
    b = (word[..., None] >> (8 * torch.arange(bits, device=c.device))) & 255
    return b.to(torch.uint8).reshape(*codes.shape[:-1], 8 * bits)


def _random_rows(n, kv_heads, key_bits, value_bits, gen):
    """Packed rows of N(0, 1) keys and values: their codes and their norms near 1 (512 in the format)."""
    dev = gen.device
    parts = []
    for bits in (key_bits, value_bits):
        cent = torch.tensor(CENTROIDS[bits], dtype=torch.float32, device=dev) / 32768
        x = torch.randn((n, kv_heads, D), generator=gen, device=dev)
        parts.append(_pack(torch.bucketize(x, (cent[1:] + cent[:-1]) / 2), bits))
    norms = (512 + 45 * torch.randn((n, kv_heads, 2), generator=gen, device=dev)).round().clamp(1, 32767)
    norms = norms.to(torch.int32)
    parts.append(torch.stack((norms & 255, norms >> 8), -1).to(torch.uint8).reshape(n, kv_heads, 4))
    return torch.cat(parts, -1)


def _cache(case, lengths, rows, spare=0):
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    pc = PagedCache(QuantConfig(key_bits=case["key_bits"], value_bits=case["value_bits"]),
                    geo=Geometry(case["kv_heads"], case.get("groups", 4), D), max_seqs=len(lengths) + spare,
                    capacity=max(lengths), page_tokens=PAGE)
    pc.put_rows(list(range(len(lengths))), lengths, rows)
    return pc


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab + case["pad"]), generator=gen, device="cuda") * 2.5
        # a few likely tokens in each row, as a trained model gives
        at = torch.randint(vocab, (rows, 24), generator=gen, device="cuda")
        x.scatter_add_(1, at, 4 * torch.rand((rows, 24), generator=gen, device="cuda") + 4)
        s["logits"] = x.to(getattr(torch, case["dtype"]))[:, :vocab]
        s["uniform"] = torch.rand((rows, vocab), generator=gen, device="cuda")
        s["settings"] = {k: v.cuda() for k, v in _settings(case).items()}
        if own:
            from insitu_b200.sampling import Sampler
            s["sampler"] = Sampler(**s["settings"])
        return s
    lengths = [t + case["nodes"] for t in _contexts(case)]
    s["lengths"] = lengths
    rows = _random_rows(sum(lengths), case["kv_heads"], case["key_bits"], case["value_bits"], gen)
    if case["op"] == "tree":
        heads = case["kv_heads"] * case["groups"]
        q = torch.randn((case["batch"] * case["nodes"], heads, D), generator=gen, device="cuda") / 4
        s["q"] = (q * 65536).round().to(torch.int32)
        s["parents"] = _parents(case)
        if own:
            from insitu_b200.tree import DraftTree
            s["cache"] = _cache(case, lengths, rows)
            s["tree"] = DraftTree(s["parents"])
            s["seqs"] = list(range(case["batch"]))
            return s
        s["rows"] = _padded(rows, lengths)
        s["contexts"] = torch.tensor(_contexts(case), device="cuda")
        s["seen"] = _seen(s["parents"], torch.device("cuda"))
        return s
    s["kept"] = _kept(case, seed)
    batch = case["batch"]
    if own:
        s["cache"] = _cache(case, lengths, rows, spare=batch)
        return s
    # a paged pool of whole rows, each sequence's pages in order, and room for the forks
    per_seq = -(-max(lengths) // PAGE)
    pool = torch.zeros((2 * batch * per_seq * PAGE, *rows.shape[1:]), dtype=torch.uint8, device="cuda")
    table = torch.arange(2 * batch * per_seq, device="cuda").reshape(2 * batch, per_seq)
    length = torch.tensor(lengths, device="cuda")
    seq = torch.repeat_interleave(torch.arange(batch, device="cuda"), length)
    pos = torch.arange(len(seq), device="cuda") - torch.repeat_interleave(length.cumsum(0) - length, length)
    pool[table[seq, pos // PAGE] * PAGE + pos % PAGE] = rows
    s.update(pool=pool, table=table)
    return s


def _settings(case):
    """Sampling settings of each row; a filter that is off has its neutral value."""
    n, f = case["rows"], case["filters"]
    rng = random.Random(n + 31 * case["vocab"])
    temperature, top_k, top_p, min_p = [], [], [], []
    for i in range(n):
        on = rng.choice(("k", "p", "m", "kp", "kpm", "pm", "", "kp")) if f == "mixed" else f.replace("none", "")
        temperature.append(0.0 if f == "mixed" and i % 16 == 5 else rng.choice((0.6, 0.7, 0.8, 1.0)))
        top_k.append(rng.choice((1, 20, 50, 200)) if "k" in on else 0)
        top_p.append(rng.choice((0.8, 0.9, 0.95)) if "p" in on else 1.0)
        min_p.append(rng.choice((0.02, 0.05, 0.1)) if "m" in on else 0.0)
    return {"temperature": torch.tensor(temperature), "top_k": torch.tensor(top_k, dtype=torch.int32),
            "top_p": torch.tensor(top_p), "min_p": torch.tensor(min_p)}


def _padded(rows, lengths):
    """Rows of all sequences, one after another -> (batch, longest, heads, bytes), zeros after each one's last."""
    length = torch.tensor(lengths, device=rows.device)
    pos = torch.arange(max(lengths), device=rows.device)
    inside = pos < length[:, None]
    out = torch.zeros((len(lengths), max(lengths), *rows.shape[1:]), dtype=torch.uint8, device=rows.device)
    out[inside] = rows
    return out


def _seen(parents, device):
    """(batch, nodes, nodes) truth values: node j is node i or one of its ancestors."""
    out = torch.zeros((len(parents), len(parents[0]), len(parents[0])), dtype=torch.bool)
    for b, tree in enumerate(parents):
        for i, p in enumerate(tree):
            if p >= 0:
                out[b, i] = out[b, p]
            out[b, i, i] = True
    return out.to(device)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"tree": _plain_tree, "pages": _plain_pages, "sample": _plain_sample}[case["op"]](case, state)


def _run_own(case, s):
    if case["op"] == "tree":
        return s["cache"].tree_scan(s["seqs"], s["q"], s["tree"])
    if case["op"] == "sample":
        return s["sampler"](s["logits"], s["uniform"])
    pc, batch = s["cache"], case["batch"]
    forks = list(range(batch, 2 * batch))
    base = [case["context"]] * batch if case["kind"] == "accept" else [0] * batch
    first = base[0] // PAGE * PAGE                 # the first row of the page that holds row `base`
    pc.fork(list(range(batch)), forks)
    pc.compact(forks, s["kept"], base)
    rows = pc.rows(forks, first, base[0] + case["keep"] - first)
    pc.truncate(forks, 0)
    return rows


def _decode(rows, centroids, first_byte, bits, norms):
    """Codes at `first_byte` of packed rows (..., bytes) -> centroid times norm, (..., 64) float32."""
    j = torch.arange(D, device=rows.device) * bits
    lo = rows[..., first_byte + j // 8].to(torch.int32)
    hi = rows[..., torch.clamp(first_byte + j // 8 + 1, max=rows.shape[-1] - 1)].to(torch.int32)
    codes = ((lo | (hi << 8)) >> (j % 8)) & ((1 << bits) - 1)
    table = torch.tensor(centroids, dtype=torch.float32, device=rows.device) / 32768
    return table[codes] * (norms[..., None] / 512)


def _plain_tree(case, s):
    kb, vb, h, n = case["key_bits"], case["value_bits"], case["kv_heads"], case["nodes"]
    rows, batch, g = s["rows"], case["batch"], case["groups"]
    at = 8 * (kb + vb)
    norm = rows[..., at:].contiguous().view(torch.int16).to(torch.float32)
    k = _decode(rows, CENTROIDS[kb], 0, kb, norm[..., 0]).transpose(1, 2)
    v = _decode(rows, CENTROIDS[vb], 8 * kb, vb, norm[..., 1]).transpose(1, 2)
    q = (s["q"].to(torch.float32) / 65536).reshape(batch, n, h, g, D).permute(0, 2, 1, 3, 4)
    score = q.reshape(batch, h, n * g, D) @ k.transpose(2, 3)
    pos = torch.arange(rows.shape[1], device=rows.device)
    node = pos - s["contexts"][:, None]
    inside = (node >= 0) & (node < n)
    drafted = s["seen"].gather(2, node.clamp(0, n - 1)[:, None].expand(-1, n, -1))
    seen = (node < 0)[:, None] | (inside[:, None] & drafted)
    seen = seen.repeat_interleave(g, 1)[:, None]
    score = torch.where(seen, score, float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    return out.reshape(batch, h, n, g, D).permute(0, 2, 1, 3, 4).reshape(batch * n, h * g, D).to(torch.bfloat16)


def _plain_pages(case, s):
    pool, table, batch = s["pool"], s["table"], case["batch"]
    base = case["context"] if case["kind"] == "accept" else 0
    full, first = (case["context"] + case["nodes"]) // PAGE, base // PAGE * PAGE
    keep = s["kept"].cuda()
    # fork: whole pages are shared; a page that is not full, or that the fork writes, becomes its own
    forked = torch.cat((table[:batch, :first // PAGE], table[batch:, first // PAGE:]), 1)
    if case["kind"] == "accept":
        pages = min(table.shape[1], full + 1)
        old, new = table[:batch, first // PAGE:pages], forked[:, first // PAGE:pages]
        paged = pool.view(-1, PAGE, *pool.shape[1:])
        paged[new.reshape(-1)] = paged[old.reshape(-1)]
        source = forked
    else:
        source = table[:batch]
    seq = torch.arange(batch, device="cuda")[:, None]
    src = base + keep
    dst = base + torch.arange(case["keep"], device="cuda").expand_as(keep)
    pool[forked[seq, dst // PAGE] * PAGE + dst % PAGE] = pool[source[seq, src // PAGE] * PAGE + src % PAGE]
    pos = torch.arange(first, base + case["keep"], device="cuda").expand(batch, -1)
    out = pool[forked[seq, pos // PAGE] * PAGE + pos % PAGE]
    return out.reshape(-1, *pool.shape[1:])


def _plain_sample(case, s):
    x = s["logits"].to(torch.float32)
    x = torch.where(torch.isnan(x), float("-inf"), x)
    t, k, top_p, min_p = (s["settings"][name][:, None] for name in ("temperature", "top_k", "top_p", "min_p"))
    vocab = x.shape[1]
    greedy = t == 0
    x, index = torch.sort(x, dim=1, descending=True, stable=True)
    z = x / torch.where(greedy, 1.0, t)
    z = z - z[:, :1]
    rank = torch.arange(vocab, device=x.device)
    keep = (x > float("-inf")) & (rank < torch.where(k > 0, k, vocab))
    w = torch.where(keep, torch.exp(z), 0.0)
    upto = torch.cumsum(w, 1)
    keep &= (upto - w < top_p * upto[:, -1:]) | (top_p >= 1)
    keep &= w >= min_p
    keep &= ~greedy | (rank == 0)
    key = z - torch.log(-torch.log(s["uniform"].gather(1, index)))
    key = torch.where(keep, key, float("-inf"))
    best = key == key.amax(1, keepdim=True)
    token = torch.where(best & keep, index, vocab).amin(1)
    chosen = torch.where(index == token[:, None], z, float("-inf")).amax(1)
    mass = torch.where(keep, w, 0.0).sum(1)
    return token, chosen - torch.log(mass)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------

def work(case):
    if case["op"] == "tree":
        row = 8 * (case["key_bits"] + case["value_bits"]) + 4
        heads = case["kv_heads"] * case["groups"]
        pairs = 0
        for t, tree in zip(_contexts(case), _parents(case)):
            depth = []
            for p in tree:
                depth.append(1 if p < 0 else depth[p] + 1)
            pairs += t * len(tree) + sum(depth)
        total = sum(_contexts(case)) + case["batch"] * case["nodes"]
        vectors = case["batch"] * case["nodes"] * heads * D
        return {"bytes": total * case["kv_heads"] * row + vectors * (4 + 2), "flops": 4 * D * heads * pairs}
    if case["op"] == "pages":
        row = case["kv_heads"] * (8 * (case["key_bits"] + case["value_bits"]) + 4)
        base = case["context"] if case["kind"] == "accept" else 0
        # the fork's own page, the rows that move, the rows that come back: read and written once each
        moved = base % PAGE + case["keep"]
        return {"bytes": case["batch"] * row * (2 * moved + 2 * moved), "flops": 0}
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[case["dtype"]]
    values = case["rows"] * case["vocab"]
    # a filtered row needs the random numbers of the few tokens that it keeps only
    return {"bytes": values * size + (4 * values if case["filters"] == "none" else 0) + 12 * case["rows"],
            "flops": 4 * values}


def exact(case, seed):
    s = prepare(case, seed) if not own else None
    if s is None or case["op"] == "pages":
        return None
    if case["op"] == "sample":
        return None, _exact_logprob(case, s)
    kb, vb, n, g = case["key_bits"], case["value_bits"], case["nodes"], case["groups"]
    out = torch.zeros((case["batch"] * n, case["kv_heads"] * g, D), dtype=torch.float64, device="cuda")
    weights = {b: (1 << torch.arange(b, device="cuda")).double() for b in (kb, vb)}
    for b, length in enumerate(s["lengths"]):
        context = length - n
        for h in range(case["kv_heads"]):
            rows = s["rows"][b, :length, h]
            bits = ((rows[:, :, None] >> torch.arange(8, device="cuda")) & 1).reshape(length, -1)
            norm = rows[:, -4:].long()
            signed = lambda lo, hi: ((lo + 256 * hi + 32768) % 65536 - 32768).double() / 512  # noqa: E731

            def vectors(first, width, scale):
                code = (bits[:, first:first + D * width].reshape(length, D, width).double() @ weights[width]).long()
                return torch.tensor(CENTROIDS[width], dtype=torch.float64, device="cuda")[code] / 32768 * scale[:, None]

            key = vectors(0, kb, signed(norm[:, 0], norm[:, 1]))
            value = vectors(D * kb, vb, signed(norm[:, 2], norm[:, 3]))
            for i0 in range(0, n, 8):
                i1 = min(n, i0 + 8)
                q = s["q"][b * n + i0:b * n + i1, h * g:(h + 1) * g].double() / 65536
                score = q @ key.T
                for i in range(i0, i1):
                    path, j = [], i
                    while j >= 0:
                        path.append(j)
                        j = s["parents"][b][j]
                    hidden = [context + j for j in range(n) if j not in path]
                    score[i - i0][:, hidden] = float("-inf")
                out[b * n + i0:b * n + i1, h * g:(h + 1) * g] = torch.softmax(score, -1) @ value
    return out


def _exact_logprob(case, s):
    """The log-probability of each row's token, row by row on the CPU's doubles."""
    x, u = s["logits"].double().cpu(), s["uniform"].double().cpu()
    got = torch.zeros(len(x), dtype=torch.float64)
    for r in range(len(x)):
        t, k, top_p, min_p = (float(s["settings"][name][r]) for name in ("temperature", "top_k", "top_p", "min_p"))
        if t == 0:
            continue
        order = torch.argsort(x[r], descending=True, stable=True)
        if k > 0:
            order = order[:int(k)]
        weight = torch.exp((x[r][order] - x[r][order[0]]) / t)
        if top_p < 1:
            share = torch.cumsum(weight, 0) / weight.sum()
            last = int(torch.searchsorted(share, torch.tensor(top_p, dtype=torch.float64)))
            order, weight = order[:last + 1], weight[:last + 1]
        stays = weight >= min_p
        order, weight = order[stays], weight[stays]
        race = -torch.log(u[r][order]) / weight
        won = int(torch.argmin(race))
        got[r] = torch.log(weight[won] / weight.sum())
    return got.cuda()
