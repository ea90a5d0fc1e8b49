"""Rotated appends, a cache held in 4 bits and its attention, and log probabilities: what is measured, on which shapes.

Four operators of a serving loop, each in its plain form (elementary torch operations in 32 bits, angles in 64) and as
the calls of ``CUDABackend``:

* ``append``  new queries and keys turned by their positions, keys and values written to their pages
* ``chunk``   a prompt's chunk turned and written to pages of 4 bits a value, and all rows read back for its attention
* ``paged``   attention of one new token per sequence over pages of 4 bits a value
* ``score``   log probabilities of given tokens, the entropy and the most likely tokens of rows of logits

A row of 4-bit pages holds dim / 2 bytes of codes (the even dim in the low half) and, for each 32 values, two float16
numbers s and z: code c stands for s (64 + c) + z, rounded to float16.  Head counts and dims are those of this package's
model configurations (``synthetic.py``) and a few others.
"""
import functools
import importlib
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_GROUP = 32   # values that share s and z


def listed():
    """The measured cases.  spread -1: every sequence as long as `length`; else seeds its lengths.  window 0: none."""
    return [
        # the decode step of 64 sequences at Heavy Medium's heads: queries and keys turned, one row a sequence written
        dict(name="append step", op="append", type="bf16", batch=64, heads=32, kv_heads=8, dim=128, length=4096, page=64,
             tokens=0, rotated=128, split=False, positions=False, theta=5e5, spread=1),
        # ragged flashlite prompts entering the cache
        dict(name="append prompts", op="append", type="bf16", batch=9, heads=16, kv_heads=4, dim=128, length=4096, page=32,
             tokens=1, rotated=128, split=False, positions=False, theta=5e5, spread=2),
        # flashnano-1.7 after an eviction: rows and positions differ, split-half pairs
        dict(name="append moved", op="append", type="f16", batch=24, heads=16, kv_heads=4, dim=64, length=1500, page=16,
             tokens=1, rotated=64, split=True, positions=True, theta=1e4, spread=3),
        # the second chunk of one short prompt of the smallest model into a 4-bit cache
        dict(name="chunk nano15", op="chunk", type="f32", batch=1, heads=8, kv_heads=2, dim=32, length=200, page=16,
             earlier=56, rotated=32, split=False, positions=False, theta=1e4, spread=-1),
        # a prefill batch at Heavy Medium's heads: chunks of ragged prompts behind what is there
        dict(name="chunk heavy", op="chunk", type="bf16", batch=6, heads=32, kv_heads=8, dim=128, length=2048, page=64,
             earlier=6000, rotated=128, split=False, positions=False, theta=5e5, spread=4),
        # a chat of the smallest model, float32 queries: a call's latency counts
        dict(name="paged nano15 one", op="paged", type="f32", batch=1, heads=8, kv_heads=2, dim=32, length=256, page=16,
             window=64, sinks=4, weights=False, spread=-1),
        # one user's long document at Heavy Medium's heads: the whole GPU works on one sequence
        dict(name="paged heavy long", op="paged", type="bf16", batch=1, heads=32, kv_heads=8, dim=128, length=32768,
             page=64, window=0, sinks=0, weights=False, spread=-1),
        # a flashlite batch whose cache will be evicted: every row's weight is added up
        dict(name="paged lite weights", op="paged", type="f16", batch=24, heads=16, kv_heads=4, dim=128, length=8192,
             page=32, window=0, sinks=0, weights=True, spread=5),
        # a full server at Heavy Medium's heads, contexts to 32768: what 4 bits make room for
        dict(name="paged heavy batch", op="paged", type="bf16", batch=32, heads=32, kv_heads=8, dim=128, length=32768,
             page=64, window=0, sinks=0, weights=False, spread=6),
        # one sequence's next token, with its alternatives
        dict(name="score one", op="score", type="f32", rows=1, vocab=64000, given=1, top=20),
        # a decode batch, logits in 16 bits
        dict(name="score batch", op="score", type="bf16", rows=64, vocab=64000, given=1, top=20),
        # all tokens of flashnano prompts scored: the reference's return_all logits
        dict(name="score prompts", op="score", type="f32", rows=4096, vocab=32000, given=2, top=5),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    """One more case: any of the operators, types and head layouts, lengths and batches over their logarithm."""
    op = rng.choice(["paged", "paged", "score", "score", "append", "chunk"])
    case = dict(op=op, type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if op == "score":
        vocab = _log(rng, 50, 200000)
        return dict(case, vocab=vocab, rows=_log(rng, 1, max(1, min(4096, (1 << 27) // vocab))),
                    given=rng.choice([0, 1, 1, 2, 5]), top=min(vocab, rng.choice([0, 1, 5, 20, _log(rng, 1, 64)])))
    heads, kv_heads, dim = rng.choice([(8, 2, 32), (16, 4, 64), (16, 8, 64), (16, 4, 128), (32, 8, 128), (12, 12, 96),
                                       (20, 2, 64), (9, 3, 32), (5, 1, 96), (6, 2, 128), (16, 1, 64)])
    if op == "append" and rng.random() < 0.3:
        heads, kv_heads, dim = rng.choice([(4, 2, 16), (6, 2, 40), (5, 1, 80), (9, 3, 24)])
    case.update(heads=heads, kv_heads=kv_heads, dim=dim, spread=rng.choice([-1] + [rng.randrange(1, 1 << 20)] * 3))
    if op == "paged":
        length = _log(rng, 1, 32768)
        row = kv_heads * dim * 5 // 8
        return dict(case, length=length, batch=_log(rng, 1, max(1, min(64, (300 << 20) // (row * length)))),
                    page=rng.choice([1, 8, 16, 20, 32, 64, 128]), window=rng.choice([0, 0, _log(rng, 1, length)]),
                    sinks=rng.choice([0, _log(rng, 1, 100)]), weights=rng.random() < 0.3)
    rotated = rng.choice([dim, dim, dim // 2 // 2 * 2])
    case.update(rotated=rotated, split=rng.random() < 0.5, positions=rng.random() < 0.4, theta=rng.choice([1e4, 5e5]),
                page=rng.choice([1, 8, 16, 20, 32, 64, 128]))
    if op == "append":
        length = _log(rng, 1, 4096)
        return dict(case, length=length, batch=_log(rng, 1, max(1, min(64, 30000 // length))), tokens=rng.choice([0, 1]))
    length = _log(rng, 1, 2048)
    earlier = rng.choice([0, _log(rng, 1, 6000)])
    return dict(case, length=length, earlier=earlier, batch=_log(rng, 1, max(1, min(40, 30000 // (length + earlier)))))


def _lengths(case):
    """The sequences' lengths, or those of their chunks, from the case alone."""
    if case["spread"] < 0:
        return [case["length"]] * case["batch"]
    rng = random.Random(case["spread"])
    found = [rng.randint(1, case["length"]) for _ in range(case["batch"])]
    found[rng.randrange(len(found))] = case["length"]
    return found


def _rows(case):
    """New rows and all rows of each sequence, of an append or a chunk."""
    lengths, rng = _lengths(case), random.Random(case["spread"] + 1)
    if case["op"] == "chunk":
        return lengths, [n + (rng.randint(0, case["earlier"]) if case["spread"] >= 0 else case["earlier"]) for n in lengths]
    if not case["tokens"]:
        return [1] * len(lengths), lengths
    return [rng.randint(0, n) for n in lengths[:-1]] + [lengths[-1]], lengths


def _offsets(counts):
    total = [0]
    for n in counts:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device="cuda")


def _table(lengths, page, gen):
    """A page table [batch, pages] of shuffled pages, -1 behind each sequence's last; and the pages used."""
    need = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(need), generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, max(sum(need), 1)


def _packed(pages, case, gen):
    """Pages of 4 bits with rows as a model leaves them: random codes, steps around 0.25, values around 0.  A head's rows
    of a page lie one behind the other."""
    kv, page, dim = case["kv_heads"], case["page"], case["dim"]
    pool = torch.randint(0, 256, (pages, kv, page, dim * 5 // 8), generator=gen, device="cuda", dtype=torch.uint8)
    step = (torch.rand(pages, kv, page, dim // _GROUP, generator=gen, device="cuda") * 0.2 + 0.15).half()
    base = (torch.randn(step.shape, generator=gen, device="cuda") * 0.1 - 71.5 * step.float()).half()
    pool[..., dim // 2:] = torch.stack([step, base], -1).flatten(-2).contiguous().view(torch.uint8)
    return pool.permute(0, 2, 1, 3)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = _TYPES[case["type"]]

    def rand(*shape, scale=1.0):
        return torch.randn(shape, generator=gen, device="cuda", dtype=kind) * scale

    state = dict(case=case)
    if case["op"] == "score":
        rows, vocab = case["rows"], case["vocab"]
        # logits of a trained model: a broad floor, and a few dozen tokens well above it
        logits = rand(rows, vocab, scale=2.0)
        likely = torch.rand(rows, vocab, generator=gen, device="cuda", dtype=kind)
        logits += torch.where(likely < 24 / vocab, likely * (vocab / 2), 0.0)
        tokens = torch.randint(0, vocab, (rows, case["given"]), generator=gen, device="cuda", dtype=torch.int32)
        tokens[torch.rand(tokens.shape, generator=gen, device="cuda") < 0.02] = -1   # the padding of a batch
        state.update(logits=logits, tokens=tokens)
        return state
    kv, dim, page, heads = case["kv_heads"], case["dim"], case["page"], case["heads"]
    new, lengths = (None, _lengths(case)) if case["op"] == "paged" else _rows(case)
    table, pages = _table(lengths, page, gen)
    state.update(table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    if case["op"] == "append":
        state.update(key_pages=rand(pages, page, kv, dim), value_pages=rand(pages, page, kv, dim))
    else:
        state.update(key_pages=_packed(pages, case, gen), value_pages=_packed(pages, case, gen))
    if case["op"] == "paged":
        state["query"] = rand(case["batch"], heads, dim, scale=1.5)
        if case["weights"]:
            state["weights"] = torch.zeros(case["batch"], kv, table.shape[1] * page, device="cuda")
        return state
    n = sum(new)
    state.update(query=rand(n, heads, dim, scale=1.5), keys=rand(n, kv, dim), values=rand(n, kv, dim), offsets=_offsets(new))
    if case["op"] == "append" and not case["tokens"]:
        state["offsets"] = None
    half = case["rotated"] // 2
    state["frequencies"] = (case["theta"] ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)).float()
    state["positions"] = None
    if case["positions"]:   # rows were given up before these: positions run ahead of the rows
        ahead = torch.randint(0, 20000, (n,), generator=gen, device="cuda")
        state["positions"] = (torch.arange(n, device="cuda") + ahead).to(torch.int32)
    if case["op"] == "chunk":
        state["all_offsets"] = _offsets(lengths)
        state.update(all_keys=torch.empty(sum(lengths), kv, dim, device="cuda", dtype=kind),
                     all_values=torch.empty(sum(lengths), kv, dim, device="cuda", dtype=kind))
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _places(s):
    """Sequence and row of each new token."""
    lengths, i = s["lengths"].long(), torch.arange(s["keys"].shape[0], device="cuda")
    if s["offsets"] is None:
        return i, lengths - 1
    offsets = s["offsets"].long()
    sequence = torch.searchsorted(offsets, i, right=True) - 1
    return sequence, lengths[sequence] - offsets[sequence + 1] + i


def _turned(x, position, frequencies, split):
    """The first 2 n dims of x [tokens, heads, dim] turned, in 32 bits; angles and their sines in 64."""
    n = len(frequencies)
    angle = position.double()[:, None] * frequencies.double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = x.float().clone()
    a, b = (x[..., :n], x[..., n:2 * n]) if split else (x[..., :2 * n:2], x[..., 1:2 * n:2])
    first, second = a * cos - b * sin, b * cos + a * sin
    if split:
        x[..., :n], x[..., n:2 * n] = first, second
    else:
        x[..., :2 * n:2], x[..., 1:2 * n:2] = first, second
    return x


def _quantised(x):
    """Rows [.., dim] in 32 bits as bytes of 4-bit pages."""
    groups = x.unflatten(-1, (-1, _GROUP))
    low, high = groups.amin(-1), groups.amax(-1)
    step = ((high - low) * (1 / 15)).half()
    base = (low - 64 * step.float()).half()
    held = torch.isfinite(step) & torch.isfinite(base)
    step, base = (torch.where(held, y, math.nan) for y in (step, base))
    code = (torch.round((groups - base.float()[..., None]) / step.float()[..., None]) - 64).clamp(0, 15)
    code = torch.where(held[..., None] & (step != 0)[..., None], code, 0).to(torch.uint8).flatten(-2)
    return torch.cat([code[..., ::2] | code[..., 1::2] << 4,
                      torch.stack([step, base], -1).flatten(-2).contiguous().view(torch.uint8)], -1)


def _values(rows):
    """What rows [.., bytes] of 4-bit pages stand for, in 32 bits."""
    dim = rows.shape[-1] * 8 // 5
    codes = rows[..., :dim // 2]
    code = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).unflatten(-1, (-1, _GROUP)).float()
    pair = rows[..., dim // 2:].contiguous().view(torch.float16).unflatten(-1, (-1, 2)).float()
    return (pair[..., :1] * (64 + code) + pair[..., 1:]).half().float().flatten(-2)


def _plain_append(s):
    case, table = s["case"], s["table"]
    sequence, row = _places(s)
    position = row if s["positions"] is None else s["positions"].long()
    query, keys = (_turned(s[x], position, s["frequencies"], case["split"]) for x in ("query", "keys"))
    ids, at = table[sequence, row // case["page"]].long(), row % case["page"]
    if case["op"] == "append":
        s["key_pages"][ids, at] = keys.to(s["keys"].dtype)
        s["value_pages"][ids, at] = s["values"]
        return [query.to(s["query"].dtype), s["key_pages"], s["value_pages"]]
    s["key_pages"][ids, at] = _quantised(keys)
    s["value_pages"][ids, at] = _quantised(s["values"].float())
    i, offsets = torch.arange(s["all_keys"].shape[0], device="cuda"), s["all_offsets"].long()
    sequence = torch.searchsorted(offsets, i, right=True) - 1
    row = i - offsets[sequence]
    ids, at = table[sequence, row // case["page"]].long(), row % case["page"]
    s["all_keys"].copy_(_values(s["key_pages"][ids, at]))
    s["all_values"].copy_(_values(s["value_pages"][ids, at]))
    return [query.to(s["query"].dtype), s["all_keys"], s["all_values"]]


def _seen(lengths, row, window, sinks):
    """Whether each sequence's newest token sees the row."""
    position = lengths[:, None] - 1
    seen = row <= position
    return seen & ((position - row < window) | (row < sinks)) if window else seen


def _plain_paged(s):
    case, table = s["case"], s["table"]
    b, h, d = s["query"].shape
    kv, page = case["kv_heads"], case["page"]
    capacity = table.shape[1] * page
    row = torch.arange(capacity, device="cuda")
    visible = _seen(s["lengths"].long(), row, case["window"], case["sinks"])
    out = torch.empty(b, h, d, device="cuda")
    for i in range(0, b, 8):   # eight sequences at a time: the rows in 32 bits take much memory
        part = slice(i, i + 8)
        ids = table[part][:, row // page].clamp_min(0).long()
        k, v = (_values(s[x][ids, row % page]).permute(0, 2, 1, 3) for x in ("key_pages", "value_pages"))
        q = s["query"][part].float().reshape(-1, kv, h // kv, d)
        e = (q @ k.transpose(-1, -2)) / math.sqrt(d)
        e = e.masked_fill(~visible[part][:, None, None], -math.inf)
        e = torch.exp(e - e.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min))
        p = e / e.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
        out[part] = (p @ v).reshape(-1, h, d)
        if case["weights"]:
            s["weights"][part] += p.sum(2)
    out = out.to(s["query"].dtype)
    return [out, s["weights"]] if case["weights"] else [out]


def _plain_score(s):
    case, tokens = s["case"], s["tokens"].long()
    parts = []
    for i in range(0, case["rows"], 512):
        x = s["logits"][i:i + 512].float()
        t = tokens[i:i + 512]
        shifted = x - x.amax(-1, keepdim=True)
        e = torch.exp(shifted)
        total = e.sum(-1, keepdim=True)
        log_p = shifted - torch.log(total)
        inside = (t >= 0) & (t < case["vocab"])
        given = torch.where(inside, log_p.gather(1, t.clamp(0, case["vocab"] - 1)), 0.0)
        entropy = torch.log(total[:, 0]) - (e * shifted.clamp_min(-1e30)).sum(-1) / total[:, 0]
        order = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :case["top"]]
        parts.append((given, entropy, order.to(torch.int32), log_p.gather(1, order)))
    return [torch.cat(p) for p in zip(*parts)]


# ---- the framework's calls ----------------------------------------------------------------------------------------
@functools.cache
def _backend_of(stream):
    now = torch.cuda.current_stream()
    package = importlib.import_module("miraclereasoning-cpu_b200")
    return package.CUDABackend(device_index=now.device_index, stream=now.cuda_stream)


def _backend():
    """The program's backend of the device and the stream that torch works on at this call."""
    return _backend_of(torch.accelerator.current_stream())


def _own_append(s):
    case = s["case"]
    query = _backend().append_rotated(s["keys"], s["values"], s["key_pages"], s["value_pages"], s["table"], s["lengths"],
                                      s["frequencies"], s["offsets"], positions=s["positions"], query=s["query"],
                                      split_half=case["split"])
    if case["op"] == "append":
        return [query, s["key_pages"], s["value_pages"]]
    return [query, *_backend().read_pages(s["key_pages"], s["value_pages"], s["table"], s["lengths"], s["all_offsets"],
                                          s["all_keys"], s["all_values"])]


def _own_paged(s):
    case, weights = s["case"], s.get("weights")
    out = _backend().paged_attention(s["query"], s["key_pages"], s["value_pages"], s["table"], s["lengths"],
                                     window=case["window"] or None, sinks=case["sinks"], weights=weights)
    return [out] if weights is None else [out, weights]


def _own_score(s):
    return list(_backend().log_probabilities(s["logits"], s["tokens"], top=s["case"]["top"]))


def run(state):
    op = state["case"]["op"]
    if own:
        return {"paged": _own_paged, "score": _own_score}.get(op, _own_append)(state)
    return {"paged": _plain_paged, "score": _plain_score}.get(op, _plain_append)(state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def work(case):
    size = _BYTES[case["type"]]
    if case["op"] == "score":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + case["rows"] * (8 * case["given"] + 4 + 8 * case["top"]), "flops": 5.0 * n}
    kv, dim, heads = case["kv_heads"], case["dim"], case["heads"]
    packed = kv * dim * 5 // 8
    if case["op"] == "paged":
        seen = 0
        for n in _lengths(case):
            window = case["window"]
            seen += n if not window or n <= window else min(n, window + min(case["sinks"], n - window))
        total = 2 * seen * packed + 2 * case["batch"] * heads * dim * size
        return {"bytes": total + (8 * seen * kv if case["weights"] else 0), "flops": 4.0 * seen * heads * dim}
    new, lengths = _rows(case)
    n, m = sum(new), sum(lengths)
    total = 2 * n * heads * dim * size + 2 * n * kv * dim * size   # queries in and out, keys and values in
    flops = 3.0 * n * (heads + kv) * case["rotated"]
    if case["op"] == "append":
        return {"bytes": total + 2 * n * kv * dim * size, "flops": flops}
    # the chunk's rows written in 4 bits; of those read back, the earlier ones read and all written
    return {"bytes": total + 2 * n * packed + 2 * (m - n) * packed + 2 * m * kv * dim * size, "flops": flops}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------
def _read64(row_bytes, dim):
    """Rows of 4-bit pages [rows, bytes], value by value's definition."""
    out = torch.empty(len(row_bytes), dim, dtype=torch.float64, device=row_bytes.device)
    words = row_bytes[:, dim // 2:].contiguous().view(torch.float16).double()
    for j in range(dim):
        code = (row_bytes[:, j // 2] >> (4 * (j % 2))) & 15
        g = j // 32
        out[:, j] = (words[:, 2 * g] * (code.double() + 64) + words[:, 2 * g + 1]).half().double()
    return out


def _paged64(case, s):
    outs, window, sinks = [], case["window"], case["sinks"]
    h, kv, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]
    totals = torch.zeros(case["batch"], kv, s["table"].shape[1] * page, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        ids = [i for i in s["table"][b].tolist() if i >= 0]
        rows = torch.arange(n, device="cuda")
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        if window:
            keep = (rows > n - 1 - window) | (rows < sinks)
        out = torch.zeros(h, dim, dtype=torch.float64, device="cuda")
        for g in range(kv):
            k, v = (_read64(torch.cat([s[x][i, :, g] for i in ids])[:n][keep], dim) for x in ("key_pages", "value_pages"))
            q = s["query"][b, g * h // kv:(g + 1) * h // kv].double()
            p = torch.softmax(q @ k.T * dim ** -0.5, dim=1)
            out[g * h // kv:(g + 1) * h // kv] = p @ v
            totals[b, g, rows[keep]] = p.sum(0)
        outs.append(out)
    return [torch.stack(outs)] + ([totals] if case["weights"] else [])


def _turn64(x, positions, frequencies, split):
    """As products of complex numbers."""
    n = len(frequencies)
    x = x.double().clone()
    angle = positions.double()[:, None, None] * frequencies.double()
    turn = torch.complex(torch.cos(angle), torch.sin(angle))
    index = torch.arange(n, device=x.device)
    at = (index, index + n) if split else (2 * index, 2 * index + 1)
    z = torch.complex(x[..., at[0]], x[..., at[1]]) * turn
    x[..., at[0]], x[..., at[1]] = z.real, z.imag
    return x


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "paged":
        return _paged64(case, s)
    if case["op"] == "score":
        given, entropy, ids, best = [], [], [], []
        for r in range(0, case["rows"], 256):
            x = s["logits"][r:r + 256].double()
            log_p = x - torch.logsumexp(x, dim=1, keepdim=True)
            t = s["tokens"][r:r + 256].long()
            g = torch.take_along_dim(log_p, t.clamp_min(0), dim=1)
            given.append(g.masked_fill(t < 0, 0.0))
            entropy.append(torch.special.entr(torch.exp(log_p)).sum(1))
            order = torch.argsort(-x, dim=1, stable=True)[:, :case["top"]]
            ids.append(order.int())
            best.append(torch.take_along_dim(log_p, order, dim=1))
        return [torch.cat(given), torch.cat(entropy), torch.cat(ids), torch.cat(best)]
    new, lengths = _rows(case)
    rows = torch.cat([torch.arange(n - c, n, device="cuda") for c, n in zip(new, lengths)])
    positions = rows if s["positions"] is None else s["positions"]
    query = _turn64(s["query"], positions, s["frequencies"], case["split"])
    if case["op"] == "chunk":   # codes are choices of the 32-bit values: 64 bits choose others next to a border
        return [query, None, None]
    keys, pools, at = _turn64(s["keys"], positions, s["frequencies"], case["split"]), [], 0
    for pool, source in ((s["key_pages"].double(), keys), (s["value_pages"].double(), s["values"].double())):
        at = 0
        for b, (c, n) in enumerate(zip(new, lengths)):
            ids = s["table"][b].tolist()
            for lo in range((n - c) // case["page"], -(-n // case["page"])):
                first, last = max(lo * case["page"], n - c), min((lo + 1) * case["page"], n)
                if first < last:
                    pool[ids[lo], first - lo * case["page"]:last - lo * case["page"]] = \
                        source[at + first - (n - c):at + last - (n - c)]
            at += c
        pools.append(pool)
    return [query, *pools]
