"""Three more serving operators around the compressed cache, as measured cases.

What a serving loop runs besides drafted trees, page operations and the draw:

* ``chunk``: attention of a chunk of new tokens of each sequence over the paged
  compressed cache, causal, over everything or over a sliding window and the
  first few tokens (sinks); a chunk of one token is the decode form;
* ``dense``: reading cached rows back as keys and values in floating point, in
  the rotated basis that the cache holds or in the model's own;
* ``penalties``: repetition, presence and frequency penalties of the tokens so
  far, a bias, and a mask of allowed tokens, on a batch of logits.

``run`` computes a case in plain torch operations, or, where ``own`` is true,
through the package's entry points.
"""

import math
import random

import numpy as np
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
        # the next token of one short conversation under a window: nothing but latency
        dict(name="chunk token, window 256", op="chunk", batch=1, context=511, chunk=1, window=256, sinks=4,
             kv_heads=8, groups=4, key_bits=4, value_bits=2, ragged=False),
        # the next token of a full batch of long conversations, each at its own length, under a window
        dict(name="chunk token, 64 seqs, window", op="chunk", batch=64, context=32768, chunk=1, window=4096,
             sinks=4, kv_heads=8, groups=4, key_bits=4, value_bits=2, ragged=True),
        # short turns of a chat batch, odd lengths, the 3-bit variant
        dict(name="chunk 23 x 6 seqs, 3b/3b", op="chunk", batch=6, context=9001, chunk=23, window=0, sinks=0,
             kv_heads=8, groups=4, key_bits=3, value_bits=3, ragged=True),
        # prompts that fill empty caches
        dict(name="chunk 4096 x 4, no context", op="chunk", batch=4, context=0, chunk=4096, window=0, sinks=0,
             kv_heads=8, groups=4, key_bits=4, value_bits=2, ragged=False),
        # a prompt's next piece under a window and sinks
        dict(name="chunk 2048 of 32K, window", op="chunk", batch=2, context=32768, chunk=2048, window=4096,
             sinks=4, kv_heads=8, groups=4, key_bits=4, value_bits=2, ragged=False),
        # long prompts' next pieces over everything before them: bound by exponentials and products
        dict(name="chunk 2048 x 4, 32K", op="chunk", batch=4, context=32768, chunk=2048, window=0, sinks=0,
             kv_heads=8, groups=4, key_bits=4, value_bits=2, ragged=False),
        # one turn's rows handed to code that wants the model's own keys and values
        dict(name="dense 300 rows", op="dense", batch=1, rows=300, first=100, kv_heads=8, key_bits=4,
             value_bits=2, dtype="float32", rotated=False, ragged=False),
        # a batch's rows at odd lengths as they are held, for attention in the rotated basis
        dict(name="dense 16 seqs, 3b/3b, rotated", op="dense", batch=16, rows=4001, first=37, kv_heads=8,
             key_bits=3, value_bits=3, dtype="float16", rotated=True, ragged=True),
        # a long document's whole cache moved to a dense engine
        dict(name="dense 128K rows", op="dense", batch=1, rows=131072, first=0, kv_heads=8, key_bits=4,
             value_bits=2, dtype="bfloat16", rotated=False, ragged=False),
        # the next token of one sequence, penalised
        dict(name="penalties 1 x 32000", op="penalties", rows=1, vocab=32000, dtype="float32", pad=0, history=600,
             drafted=0, bias="none", mask="none"),
        # a full batch under grammars, each row with its own settings and mask
        dict(name="penalties 256 x 128000", op="penalties", rows=256, vocab=128000, dtype="bfloat16", pad=0,
             history=2048, drafted=0, bias="none", mask="row"),
        # nodes of drafted trees: rows share their sequence's tokens and add their own path's; rows of a wider buffer
        dict(name="penalties 96 x 50003, trees", op="penalties", rows=96, vocab=50003, dtype="float16", pad=61,
             history=9000, drafted=6, bias="one", mask="one"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(("chunk", "chunk", "dense", "penalties"))
    kv_heads, groups = rng.choice((1, 2, 4, 8)), rng.choice((1, 2, 4, 8))
    key_bits, value_bits = rng.choice(((4, 2), (4, 2), (3, 3)))
    if op == "chunk":
        batch, chunk = _log_int(rng, 1, 64), _log_int(rng, 1, 4096)
        # at most the largest listed case's products, and 2^18 cached tokens of 8 heads
        pairs = 4 * 2048 * 33792 * 32 // (kv_heads * groups)
        chunk = max(1, min(chunk, int((pairs / batch) ** 0.5), (1 << 18) // batch))
        most = max(1, min(pairs // (batch * chunk) - chunk, (1 << 18) * 8 // (batch * kv_heads) - chunk, 131072))
        window = rng.choice((0, 0, _log_int(rng, 1, 8192)))
        return dict(op="chunk", batch=batch, context=_log_int(rng, 1, most) - 1, chunk=chunk, window=window,
                    sinks=rng.choice((0, 1, 4, _log_int(rng, 1, 300))) if window else 0, kv_heads=kv_heads,
                    groups=groups, key_bits=key_bits, value_bits=value_bits, ragged=rng.random() < 0.7)
    if op == "dense":
        batch = _log_int(rng, 1, 64)
        most = 131072 * 8 // (batch * kv_heads * 2)        # float32 outputs stay below the largest case's
        return dict(op="dense", batch=batch, rows=_log_int(rng, 1, min(most, 131072)), first=rng.randint(0, 600),
                    kv_heads=kv_heads, key_bits=key_bits, value_bits=value_bits,
                    dtype=rng.choice(("float32", "bfloat16", "float16")), rotated=rng.random() < 0.4,
                    ragged=rng.random() < 0.7)
    return dict(op="penalties", rows=_log_int(rng, 1, 256), vocab=_log_int(rng, 300, 64000),
                dtype=rng.choice(("float32", "bfloat16", "float16")), pad=rng.choice((0, 0, 1, 8, 61)),
                history=_log_int(rng, 1, 8192) - 1, drafted=rng.choice((0, 0, 3, 8)),
                bias=rng.choice(("none", "one", "row")), mask=rng.choice(("none", "one", "row")))


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------

def _spread(case, most, least):
    """A number for each sequence: `most`, or up to it in odd steps."""
    b = case["batch"]
    if not case["ragged"]:
        return [most] * b
    return [max(least, most * (i + 1) // b - i % 5) for i in range(b)]


def _lengths(case):
    """(tokens before, tokens of the call) of each sequence."""
    if case["op"] == "chunk":
        return _spread(case, case["context"], 0), _spread(case, case["chunk"], 1)
    return [case["first"]] * case["batch"], _spread(case, case["rows"], 1)


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


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}
    if case["op"] == "penalties":
        _prepare_penalties(case, s, gen)
        return s
    before, count = _lengths(case)
    lengths = [a + b for a, b in zip(before, count)]
    # every sequence's packed rows, one sequence after another
    s["rows"] = _random_rows(sum(lengths), case["kv_heads"], case["key_bits"], case["value_bits"], gen)
    s["before"], s["count"], s["seqs"] = before, count, list(range(case["batch"]))
    if case["op"] == "chunk":
        heads = case["kv_heads"] * case["groups"]
        q = torch.randn((sum(count), heads, D), generator=gen, device="cuda") / 4
        s["q"] = (q * 65536).round().to(torch.int32)
    else:
        s["signs"] = torch.from_numpy(np.random.Generator(np.random.PCG64(0)).integers(0, 2, D) * 2.0 - 1).cuda()
    if own:
        from insitu_b200 import Geometry, PagedCache, QuantConfig
        s["cache"] = PagedCache(QuantConfig(key_bits=case["key_bits"], value_bits=case["value_bits"]),
                                geo=Geometry(case["kv_heads"], case.get("groups", 4), D), max_seqs=case["batch"],
                                capacity=max(lengths), page_tokens=PAGE)
        s["cache"].put_rows(s["seqs"], lengths, s.pop("rows"))
    return s


def _prepare_penalties(case, s, gen):
    n, vocab, rng = case["rows"], case["vocab"], random.Random(case["rows"] + 31 * case["vocab"])
    x = torch.randn((n, vocab + case["pad"]), generator=gen, device="cuda") * 2.5
    s["logits"] = x.to(getattr(torch, case["dtype"]))[:, :vocab]
    # tokens so far: a few common ones, many rare ones, as text has
    seqs = -(-n // 24) if case["drafted"] else n
    text = lambda *shape: (vocab * torch.rand(shape, generator=gen, device="cuda") ** 4).long().clamp(max=vocab - 1)  # noqa: E731
    s["tokens"] = text(seqs, case["history"])
    lengths = [max(0, case["history"] - 37 * i % (case["history"] // 2 + 1)) for i in range(seqs)]
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    s["prompts"] = torch.tensor([k * (i % 4) // 4 for i, k in enumerate(lengths)], dtype=torch.int32, device="cuda")
    s["of"], s["drafted"] = None, None
    if case["drafted"]:
        s["of"] = torch.arange(n, device="cuda", dtype=torch.int32) // 24
        deep = torch.randint(0, case["drafted"] + 1, (n, 1), generator=gen, device="cuda")
        s["drafted"] = torch.where(torch.arange(case["drafted"], device="cuda") < deep, text(n, case["drafted"]), -1)
    pick = lambda *values: torch.tensor([rng.choice(values) for _ in range(n)])  # noqa: E731
    s["settings"] = {"repetition": pick(1.0, 1.1, 1.3, 1.05), "presence": pick(0.0, 0.5, 1.5, -0.25),
                     "frequency": pick(0.0, 0.2, 1.0, 0.1)}
    rows = {"one": 1, "row": n}
    s["bias"] = s["mask"] = None
    if case["bias"] != "none":
        # a few tokens are pushed up or down, one is banned
        bias = torch.zeros((rows[case["bias"]], vocab), device="cuda")
        at = torch.randint(vocab, (len(bias), 40), generator=gen, device="cuda")
        bias.scatter_(1, at, 4 * torch.randn((len(bias), 40), generator=gen, device="cuda"))
        bias.scatter_(1, at[:, :1], float("-inf"))
        s["bias"] = bias
    if case["mask"] != "none":
        # a grammar allows long runs of the vocabulary or single tokens
        words = -(-vocab // 32)
        shape = (rows[case["mask"]], words)
        some = torch.randint(-2 ** 31, 2 ** 31, shape, generator=gen, device="cuda")
        runs = torch.randint(-1, 1, shape, generator=gen, device="cuda")
        s["mask"] = torch.where(torch.rand(shape, generator=gen, device="cuda") < 0.2, some, runs).to(torch.int32)
    if own:
        from insitu_b200 import Penalties
        s["penalties"] = Penalties(**{k: v.cuda() for k, v in s["settings"].items()})
    else:
        s["settings"] = {k: v.cuda() for k, v in s["settings"].items()}


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if own:
        return _run_own(case, state)
    return {"chunk": _plain_chunk, "dense": _plain_dense, "penalties": _plain_penalties}[case["op"]](case, state)


def _run_own(case, s):
    if case["op"] == "chunk":
        return s["cache"].chunk_scan(s["seqs"], s["q"], s["count"], window=case["window"] or None,
                                     sinks=case["sinks"])
    if case["op"] == "dense":
        return s["cache"].dense(s["seqs"], s["before"], s["count"], dtype=getattr(torch, case["dtype"]),
                                rotated=case["rotated"])
    return s["penalties"](s["logits"], s["tokens"], s["lengths"], prompts=s["prompts"], of=s["of"],
                          drafted=s["drafted"], bias=s["bias"], mask=s["mask"])


def _decode(rows, centroids, first_byte, bits, norms):
    """Codes at `first_byte` of packed rows (..., bytes) -> centroid times norm, (..., 64) float32."""
    j = torch.arange(D, device=rows.device) * bits
    lo = rows[..., first_byte + j // 8].to(torch.int32)
    hi = rows[..., torch.clamp(first_byte + j // 8 + 1, max=rows.shape[-1] - 1)].to(torch.int32)
    codes = ((lo | (hi << 8)) >> (j % 8)) & ((1 << bits) - 1)
    table = torch.tensor(centroids, dtype=torch.float32, device=rows.device) / 32768
    return table[codes] * (norms[..., None] / 512)


def _decode_rows(case, rows):
    """Packed rows (n, heads, bytes) -> keys and values (n, heads, 64) float32."""
    kb, vb = case["key_bits"], case["value_bits"]
    norm = rows[..., 8 * (kb + vb):].contiguous().view(torch.int16).to(torch.float32)
    return (_decode(rows, CENTROIDS[kb], 0, kb, norm[..., 0]),
            _decode(rows, CENTROIDS[vb], 8 * kb, vb, norm[..., 1]))


def _plain_chunk(case, s):
    h, g, sinks, window = case["kv_heads"], case["groups"], case["sinks"], case["window"] or 1 << 30
    rows, batch, most = s["rows"], case["batch"], max(s["count"])
    before = torch.tensor(s["before"], device=rows.device)[:, None]
    count = torch.tensor(s["count"], device=rows.device)[:, None]
    row0, query0 = (before + count).cumsum(0) - before - count, count.cumsum(0) - count
    q = s["q"].to(torch.float32) / 65536
    out = torch.empty_like(q)
    # every sequence's next `step` queries at once, as many as give 2^31 scores
    step = max(1, min(most, (1 << 31) // (batch * h * g * (max(s["before"]) + most))))
    for i in range(0, most, step):
        j = i + torch.arange(min(step, most - i), device=rows.device).expand(batch, -1)
        live = j < count
        pos = before + j
        # what they can see: the sinks, and the window of the first one on
        first = (pos[:, :1] - window + 1).clamp(min=0)
        span = min(window - 1 + j.shape[1], max(s["before"]) + i + j.shape[1])
        key_at = torch.cat((torch.arange(sinks, device=rows.device).expand(batch, -1),
                            first + torch.arange(span, device=rows.device)), 1)
        early = torch.arange(sinks + span, device=rows.device) < sinks
        held = (key_at < before + count) & ~(early & (key_at >= first))
        k, v = _decode_rows(case, rows[row0 + torch.where(held, key_at, 0)])
        x = q[torch.where(live, query0 + j, 0)].reshape(batch, -1, h, g, D)
        score = torch.einsum("bnhgd,bkhd->bhgnk", x, k)
        key_at, at = key_at[:, None], pos[:, :, None]
        seen = held[:, None] & (key_at <= at) & ((key_at > at - window) | (key_at < sinks))
        score = torch.where(seen[:, None, None], score, float("-inf"))
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        out[(query0 + j)[live]] = torch.einsum("bhgnk,bkhd->bnhgd", p, v).reshape(batch, -1, h * g, D)[live]
    return out.to(torch.bfloat16)


def _hadamard(device):
    """The 64 x 64 matrix of signs whose entry (i, j) is negative where i & j has an odd number of bits."""
    i = torch.arange(D, device=device)
    both = i[:, None] & i
    odd = sum((both >> b) & 1 for b in range(6)) & 1
    return 1.0 - 2.0 * odd


def _plain_dense(case, s):
    end = torch.tensor([a + b for a, b in zip(s["before"], s["count"])], device="cuda").cumsum(0)
    count = torch.tensor(s["count"], device="cuda")
    first = torch.repeat_interleave(end - count - (count.cumsum(0) - count), count)
    k, v = _decode_rows(case, s["rows"][first + torch.arange(len(first), device="cuda")])
    if not case["rotated"]:
        # the cache holds R x, R = H diag(signs) / 8, an orthogonal matrix
        back = (_hadamard(k.device) * s["signs"] / 8).to(torch.float32)
        k, v = k @ back, v @ back
    dtype = getattr(torch, case["dtype"])
    return k.to(dtype), v.to(dtype)


def _plain_penalties(case, s):
    x, vocab = s["logits"].to(torch.float32), case["vocab"]
    at = torch.arange(s["tokens"].shape[1], device=x.device)
    said = (at >= s["prompts"][:, None]) & (at < s["lengths"][:, None])
    asked = at < s["prompts"][:, None]
    count = torch.zeros((len(s["tokens"]), vocab), device=x.device).scatter_add_(1, s["tokens"], said.float())
    prompt = torch.zeros_like(count).scatter_add_(1, s["tokens"], asked.float())
    if s["of"] is not None:
        count, prompt = count[s["of"].long()], prompt[s["of"].long()]
    if s["drafted"] is not None:
        count = count.scatter_add(1, s["drafted"].clamp(min=0), (s["drafted"] >= 0).float())
    r, presence, frequency = (s["settings"][k][:, None] for k in ("repetition", "presence", "frequency"))
    y = torch.where(count + prompt > 0, torch.where(x > 0, x / r, x * r), x)
    y = y - frequency * count - presence * (count > 0)
    if s["bias"] is not None:
        y = y + s["bias"]
    if s["mask"] is not None:
        token = torch.arange(vocab, device=x.device)
        y = torch.where((s["mask"][:, token // 32] >> (token % 32)) & 1 > 0, y, float("-inf"))
    return y.to(s["logits"].dtype)


# ---------------------------------------------------------------------------
# what a pass cannot do without, and the definition in 64 bits
# ---------------------------------------------------------------------------

SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


def work(case):
    if case["op"] == "penalties":
        values = case["rows"] * case["vocab"]
        seqs = -(-case["rows"] // 24) if case["drafted"] else case["rows"]
        rows = {"none": 0, "one": 1, "row": case["rows"]}
        extra = 4 * rows[case["bias"]] * case["vocab"] + rows[case["mask"]] * (-(-case["vocab"] // 8))
        tokens = seqs * case["history"] + case["rows"] * case["drafted"]
        return {"bytes": 2 * values * SIZE[case["dtype"]] + 8 * tokens + extra, "flops": 2 * values}
    before, count = _lengths(case)
    row = case["kv_heads"] * (8 * (case["key_bits"] + case["value_bits"]) + 4)
    if case["op"] == "dense":
        out = 2 * case["kv_heads"] * D
        return {"bytes": sum(count) * (row + out * SIZE[case["dtype"]]),
                "flops": sum(count) * out * (1 if case["rotated"] else 7)}
    heads, window, sinks = case["kv_heads"] * case["groups"], case["window"], case["sinks"]
    pairs = rows = 0
    for b, n in zip(before, count):
        if not window:
            pairs, rows = pairs + n * b + n * (n + 1) // 2, rows + b + n
            continue
        lo = max(0, b - window + 1)                        # the first query's window
        rows += b + n - lo + min(sinks, lo)
        for p in range(b, b + n):
            first = max(0, p - window + 1)
            pairs += p + 1 - first + min(sinks, first)
    return {"bytes": rows * row + sum(count) * heads * D * (4 + 2), "flops": 4 * D * heads * pairs}


def exact(case, seed):
    if own:
        return None
    s = prepare(case, seed)
    return {"chunk": _exact_chunk, "dense": _exact_dense, "penalties": _exact_penalties}[case["op"]](case, s)


def _exact_vectors(case, rows):
    """Keys and values of packed rows in 64 bits, code by code from the rows' bits."""
    bits = ((rows[..., None] >> torch.arange(8, device=rows.device)) & 1).flatten(-2)
    norm = rows[..., -4:].long()
    out, first = [], 0
    for i, width in enumerate((case["key_bits"], case["value_bits"])):
        code = bits[..., first:first + D * width].unflatten(-1, (D, width)).long()
        code = sum(code[..., j] << j for j in range(width))
        signed = (norm[..., 2 * i] + 256 * norm[..., 2 * i + 1] + 32768) % 65536 - 32768
        level = torch.tensor(CENTROIDS[width], device=rows.device)[code]
        out.append(level.double() / 2 ** 15 * (signed.double() / 2 ** 9)[..., None])
        first += D * width
    return out


def _exact_chunk(case, s):
    g, sinks, window = case["groups"], case["sinks"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    row = query = 0
    for before, count in zip(s["before"], s["count"]):
        t = torch.arange(before + count, device="cuda")
        for h in range(case["kv_heads"]):
            k, v = _exact_vectors(case, s["rows"][row:row + before + count, h])
            for i in range(0, count, 256):
                n = min(256, count - i)
                q = s["q"][query + i:query + i + n, h * g:(h + 1) * g].double() / 2 ** 16
                p = before + i + torch.arange(n, device="cuda")[:, None]
                hidden = t > p
                if window:
                    hidden |= (t <= p - window) & (t >= sinks)
                score = (q.reshape(n * g, D) @ k.T).reshape(n, g, -1).masked_fill(hidden[:, None], float("-inf"))
                out[query + i:query + i + n, h * g:(h + 1) * g] = torch.softmax(score, -1) @ v
        row += before + count
        query += count
    return out


def _exact_dense(case, s):
    found, row = [], 0
    for before, count in zip(s["before"], s["count"]):
        found.append(_exact_vectors(case, s["rows"][row + before:row + before + count]))
        row += before + count
    out = []
    for x in (torch.cat([f[i] for f in found]) for i in range(2)):
        if not case["rotated"]:
            # six stages of sums and differences undo those of the rotation, and the signs after them
            for bit in range(6):
                x = x.unflatten(-1, (D >> (bit + 1), 2, 1 << bit))
                x = torch.stack((x[..., 0, :] + x[..., 1, :], x[..., 0, :] - x[..., 1, :]), -2).flatten(-3)
            x = x / 8 * s["signs"]
        out.append(x)
    return tuple(out)


def _exact_penalties(case, s):
    y = s["logits"].double()
    for i in range(case["rows"]):
        j = i if s["of"] is None else int(s["of"][i])
        asked, end = int(s["prompts"][j]), int(s["lengths"][j])
        said = s["tokens"][j, asked:end]
        if s["drafted"] is not None:
            said = torch.cat((said, s["drafted"][i][s["drafted"][i] >= 0]))
        r, presence, frequency = (s["settings"][k][i].double() for k in ("repetition", "presence", "frequency"))
        seen = torch.cat((said, s["tokens"][j, :asked])).unique()
        y[i, seen] = torch.where(y[i, seen] > 0, y[i, seen] / r, y[i, seen] * r)
        token, times = said.unique(return_counts=True)
        y[i, token] -= frequency * times + presence
        if s["bias"] is not None:
            y[i] += s["bias"][i % len(s["bias"])].double()
        if s["mask"] is not None:
            word = s["mask"][i % len(s["mask"])].long() & 0xffffffff
            allowed = (word[:, None] >> torch.arange(32, device="cuda")) & 1
            y[i, allowed.flatten()[:case["vocab"]] == 0] = float("-inf")
    return y
