"""The paged key-value cache and its attention: what is measured, and on which shapes.

Four operators of a serving loop, each in its plain form (elementary torch operations in 32 bits) and as the calls
of ``CUDABackend``:

* ``window``  prompt attention over packed sequences, causal, with a sliding window and first rows that stay visible
* ``paged``   attention of one new token per sequence over a paged cache, optionally adding up each row's weight
* ``append``  new key / value rows written to their pages
* ``evict``   the rows of largest accumulated weight kept and copied to other pages

Head counts and dims are those of this package's model configurations (``synthetic.py``), pages are 16 to 128 rows.
"""
import functools
import importlib
import math
import random

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    """The measured cases.  window 0: none.  spread -1: every sequence as long as `length`; else seeds its lengths."""
    return [
        # a chat of the smallest model: one sequence of the full 256-token context, float32; a call's latency counts
        dict(name="paged nano15 one", op="paged", type="f32", batch=1, heads=8, kv_heads=2, dim=32, length=256,
             page=16, window=64, sinks=4, spread=-1, weights=False),
        # one user's long document at Heavy Medium's heads: the whole GPU works on one sequence
        dict(name="paged heavy long", op="paged", type="bf16", batch=1, heads=32, kv_heads=8, dim=128, length=32768,
             page=64, window=0, sinks=0, spread=-1, weights=False),
        # a local layer of flashnano-1.7 in a batch: window 512 with sinks over ragged lengths
        dict(name="paged nano17 window", op="paged", type="bf16", batch=48, heads=16, kv_heads=4, dim=64, length=2048,
             page=16, window=512, sinks=4, spread=1, weights=False),
        # a flashlite batch whose cache will be evicted: every row's weight is added up
        dict(name="paged lite weights", op="paged", type="f16", batch=24, heads=16, kv_heads=4, dim=128, length=8192,
             page=32, window=0, sinks=0, spread=2, weights=True),
        # a full server at Heavy Medium's heads: ragged lengths to half its context
        dict(name="paged heavy batch", op="paged", type="bf16", batch=32, heads=32, kv_heads=8, dim=128, length=16384,
             page=64, window=0, sinks=0, spread=3, weights=False),
        # the decode step's append at flashlighting's 24 heads
        dict(name="append step", op="append", type="bf16", batch=64, kv_heads=24, dim=128, length=4096, page=64,
             tokens=0, spread=4),
        # ragged prompts of Heavy Medium entering the cache
        dict(name="append prompts", op="append", type="bf16", batch=9, kv_heads=8, dim=128, length=4096, page=32,
             tokens=1, spread=5),
        # short prompts of the smallest model in float32
        dict(name="window nano15 f32", op="window", type="f32", batch=7, heads=8, kv_heads=2, dim=32, length=200,
             earlier=0, window=64, sinks=4, spread=6),
        # a prefill batch of flashnano-1.7: the second chunk of ragged prompts, local layer with sinks
        dict(name="window nano17 chunk", op="window", type="bf16", batch=5, heads=16, kv_heads=4, dim=64, length=1500,
             earlier=600, window=512, sinks=4, spread=7),
        # one full flashlite context, no window: the largest product
        dict(name="window lite full", op="window", type="bf16", batch=1, heads=16, kv_heads=4, dim=128, length=8192,
             earlier=0, window=0, sinks=0, spread=-1),
        # one sequence of flashnano-1.7 brought from its whole context to half
        dict(name="evict nano17", op="evict", type="bf16", batch=1, kv_heads=4, dim=64, length=2048, page=16,
             budget=1024, sinks=4, recent=128, spread=-1),
        # a server's caches of Heavy Medium brought to 4096 rows a sequence
        dict(name="evict heavy batch", op="evict", type="bf16", batch=12, kv_heads=8, dim=128, length=20000, page=64,
             budget=4096, sinks=16, recent=512, spread=8),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.5)))))))


def draw(rng):
    """One more case: any of the operators, types and head layouts, lengths and batches over their logarithm."""
    op = rng.choice(["paged", "paged", "window", "window", "append", "evict"])
    heads, kv_heads, dim = rng.choice([(8, 2, 32), (16, 4, 64), (16, 8, 64), (16, 4, 128), (24, 24, 128), (32, 8, 128),
                                       (4, 2, 16), (6, 2, 40), (5, 1, 80), (12, 12, 96), (20, 2, 64), (9, 3, 24)])
    case = dict(op=op, type=rng.choice(["bf16", "bf16", "f16", "f32"]), heads=heads, kv_heads=kv_heads, dim=dim,
                spread=rng.choice([-1] + [rng.randrange(1, 1 << 20)] * 3))
    if op == "window":
        length = _log(rng, 1, 4000)
        batch = _log(rng, 1, max(1, min(40, 4000 // length)))
        return dict(case, batch=batch, length=length,
                    earlier=rng.choice([0, 0, _log(rng, 1, max(1, 1500 // batch))]), window=rng.choice([0, _log(rng, 1, 2000)]),
                    sinks=rng.choice([0, _log(rng, 1, 100)]))
    length = _log(rng, 1, 16384)
    width = kv_heads * dim * _BYTES[case["type"]]
    case.update(length=length, batch=_log(rng, 1, max(1, min(48, (600 << 20) // (width * length)))),
                page=rng.choice([1, 8, 16, 20, 32, 64, 128]))
    if op == "paged":
        return dict(case, window=rng.choice([0, _log(rng, 1, length)]), sinks=rng.choice([0, _log(rng, 1, 100)]),
                    weights=rng.random() < 0.4)
    del case["heads"]
    if op == "append":
        return dict(case, tokens=rng.choice([0, 1]))
    budget = _log(rng, 1, length)
    recent = rng.randrange(0, budget // 2 + 1)
    return dict(case, budget=budget, recent=recent, sinks=rng.randrange(0, min(64, budget - recent) + 1))


def _lengths(case, low=1):
    """The sequences' lengths, from the case alone."""
    if case["spread"] < 0:
        return [case["length"]] * case["batch"]
    rng = random.Random(case["spread"])
    found = [rng.randint(min(low, case["length"]), case["length"]) for _ in range(case["batch"])]
    found[rng.randrange(len(found))] = case["length"]
    return found


def _appended(case, lengths):
    """How many of each sequence's rows are new: one, or (tokens 1) a share from nothing to all of them."""
    if not case["tokens"]:
        return [1] * len(lengths)
    rng = random.Random(case["spread"] + 1)
    return [rng.randint(0, n) for n in lengths[:-1]] + [lengths[-1]]


def _offsets(counts, device="cuda"):
    total = [0]
    for n in counts:
        total.append(total[-1] + n)
    return torch.tensor(total, dtype=torch.int32, device=device)


def _prompt(case):
    """New and earlier rows of each sequence of a prompt case."""
    new = _lengths(case)
    rng = random.Random(case["spread"] + 2)
    return new, [rng.randint(0, case["earlier"]) if case["spread"] >= 0 else case["earlier"] for _ in new]


def _table(lengths, page, gen, first=0):
    """A page table [batch, pages] of shuffled pages from `first` on, -1 behind each sequence's last; and the pages used."""
    need = [-(-n // page) for n in lengths]
    ids = torch.randperm(sum(need), generator=gen, device="cuda").to(torch.int32) + first
    table = torch.full((len(need), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, n in enumerate(need):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, max(sum(need), 1)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = _TYPES[case["type"]]

    def rand(*shape, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda", dtype=kind) * scale)

    state = dict(case=case)
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "window":
        new, earlier = _prompt(case)
        keys = [a + b for a, b in zip(new, earlier)]
        state.update(query=rand(sum(new), case["heads"], dim, scale=1.5), keys=rand(sum(keys), kv, dim),
                     values=rand(sum(keys), kv, dim), query_offsets=_offsets(new), key_offsets=_offsets(keys))
        return state
    lengths, page = _lengths(case), case["page"]
    table, pages = _table(lengths, page, gen)
    state.update(table=table, lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                 key_pages=rand(pages, page, kv, dim), value_pages=rand(pages, page, kv, dim))
    capacity = table.shape[1] * page
    if case["op"] == "paged":
        state["query"] = rand(case["batch"], case["heads"], dim, scale=1.5)
        if case["weights"]:
            state["weights"] = torch.zeros(case["batch"], kv, capacity, device="cuda")
    elif case["op"] == "append":
        counts = _appended(case, lengths)
        state.update(keys=rand(sum(counts), kv, dim), values=rand(sum(counts), kv, dim))
        state["offsets"] = _offsets(counts) if case["tokens"] else None
    else:
        # accumulated weights as decoding leaves them: mostly small, some large, a few exact ties
        weights = torch.rand(case["batch"], kv, capacity, generator=gen, device="cuda") ** 4 * 8
        tied = torch.rand(case["batch"], kv, capacity, generator=gen, device="cuda") < 0.1
        weights = torch.where(tied, torch.round(weights * 8) / 8, weights)
        live = torch.arange(capacity, device="cuda") < state["lengths"][:, None]
        state["weights"] = weights * live[:, None]
        target, pages = _table([min(n, case["budget"]) for n in lengths], page, gen)
        state.update(target=target, target_keys=torch.zeros(pages, page, kv, dim, device="cuda", dtype=kind),
                     target_values=torch.zeros(pages, page, kv, dim, device="cuda", dtype=kind))
    return state


# ---- the plain forms ----------------------------------------------------------------------------------------------
def _softmax_mix(scores, visible, values):
    """Weights and their mix of scores [..., q, k] in 32 bits; a row that sees nothing gives zeros."""
    scores = scores.masked_fill(~visible, -math.inf)
    peak = scores.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = torch.exp(scores - peak)
    p = p / p.sum(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).tiny)
    return p, p @ values


def _sees(position, row, window, sinks):
    """Whether the query at `position` sees the key at `row`."""
    seen = (row <= position) & (row >= 0)
    if window:
        seen = seen & ((position - row < window) | (row < sinks))
    return seen


def _gathered(pages, table, count):
    """Rows 0 .. count-1 of every sequence's table, in 32 bits: [batch, kv_heads, rows, dim]."""
    t = torch.arange(count, device=table.device)
    page = pages.shape[1]
    ids = table[:, t // page].clamp_min(0).long()
    return pages[ids, t % page].float().permute(0, 2, 1, 3)


def _plain_paged(s):
    case, table, lengths = s["case"], s["table"], s["lengths"]
    capacity = table.shape[1] * case["page"]
    b, h, d = s["query"].shape
    kv = case["kv_heads"]
    k, v = _gathered(s["key_pages"], table, capacity), _gathered(s["value_pages"], table, capacity)
    q = s["query"].float().reshape(b, kv, h // kv, d)
    row = torch.arange(capacity, device=table.device)
    position = (lengths - 1)[:, None, None, None]
    p, out = _softmax_mix((q @ k.transpose(-1, -2)) / math.sqrt(d), _sees(position, row, case["window"], case["sinks"]), v)
    out = out.reshape(b, h, d).to(s["query"].dtype)
    if not case["weights"]:
        return [out]
    s["weights"] += p.sum(2)
    return [out, s["weights"]]


def _plain_window(s):
    case = s["case"]
    n, h, d = s["query"].shape
    m, kv = s["keys"].shape[:2]
    qo, ko = s["query_offsets"].long(), s["key_offsets"].long()
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    sq, sk = torch.searchsorted(qo, i, right=True) - 1, torch.searchsorted(ko, j, right=True) - 1
    position = i - qo[sq] + (ko[sq + 1] - ko[sq]) - (qo[sq + 1] - qo[sq])
    row = j - ko[sk]
    visible = (sq[:, None] == sk) & _sees(position[:, None], row, case["window"], case["sinks"])
    q = s["query"].float().reshape(n, kv, h // kv, d).permute(1, 2, 0, 3)
    k, v = (s[x].float().permute(1, 0, 2)[:, None] for x in ("keys", "values"))
    _, out = _softmax_mix((q @ k.transpose(-1, -2)) / math.sqrt(d), visible, v)
    return [out.permute(2, 0, 1, 3).reshape(n, h, d).to(s["query"].dtype)]


def _plain_append(s):
    page, lengths, table = s["case"]["page"], s["lengths"].long(), s["table"]
    i = torch.arange(s["keys"].shape[0], device="cuda")
    if s["offsets"] is None:
        sequence, position = i, lengths - 1
    else:
        offsets = s["offsets"].long()
        sequence = torch.searchsorted(offsets, i, right=True) - 1
        position = lengths[sequence] - offsets[sequence + 1] + i
    ids = table[sequence, position // page].long()
    s["key_pages"][ids, position % page] = s["keys"]
    s["value_pages"][ids, position % page] = s["values"]
    return [s["key_pages"], s["value_pages"]]


def _plain_evict(s):
    case, table, target, weights = s["case"], s["table"], s["target"], s["weights"]
    page, budget = case["page"], case["budget"]
    b, kv, capacity = weights.shape
    row = torch.arange(capacity, device="cuda")
    n = s["lengths"].long()[:, None, None]
    rank = weights.masked_fill(row >= n, -math.inf)
    rank = rank.masked_fill((row < n) & ((row < case["sinks"]) | (row >= n - case["recent"])), math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    order = torch.where(order < n, order, capacity)
    kept = torch.sort(order, dim=-1).values
    kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=capacity)
    lengths = s["lengths"].clamp(max=budget)
    live = kept < capacity
    to = torch.arange(budget, device="cuda").clamp(max=target.shape[1] * page - 1)
    seq, head, at = torch.nonzero(live, as_tuple=True)
    source = kept[seq, head, at]
    for_rows = table[seq, source // page].long(), source % page, head
    to_rows = target[seq, to[at] // page].long(), to[at] % page, head
    s["target_keys"][to_rows] = s["key_pages"][for_rows]
    s["target_values"][to_rows] = s["value_pages"][for_rows]
    out = torch.zeros(b, kv, target.shape[1] * page, device="cuda")
    out[seq, head, at] = weights[seq, head, source]
    return [torch.where(live, kept, -1).to(torch.int32), lengths, out, s["target_keys"], s["target_values"]]


# ---- the framework's calls ----------------------------------------------------------------------------------------
@functools.cache
def _backend_of(stream):
    now = torch.cuda.current_stream()
    package = importlib.import_module("miraclereasoning-cpu_b200")
    return package.CUDABackend(device_index=now.device_index, stream=now.cuda_stream)


def _backend():
    """The program's backend of the device and the stream that torch works on at this call."""
    return _backend_of(torch.accelerator.current_stream())   # found in 0.8 us


def _own_paged(s):
    case, weights = s["case"], s.get("weights")
    out = _backend().paged_attention(s["query"], s["key_pages"], s["value_pages"], s["table"], s["lengths"],
                                     window=case["window"] or None, sinks=case["sinks"], weights=weights)
    return [out] if weights is None else [out, weights]


def _own_window(s):
    case = s["case"]
    return [_backend().window_attention(s["query"], s["keys"], s["values"], s["query_offsets"], s["key_offsets"],
                                        window=case["window"] or None, sinks=case["sinks"])]


def _own_append(s):
    _backend().append_pages(s["keys"], s["values"], s["key_pages"], s["value_pages"], s["table"], s["lengths"],
                            s["offsets"])
    return [s["key_pages"], s["value_pages"]]


def _own_evict(s):
    case = s["case"]
    kept, lengths, weights = _backend().evict_pages(
        s["key_pages"], s["value_pages"], s["table"], s["lengths"], s["weights"], s["target"], budget=case["budget"],
        sinks=case["sinks"], recent=case["recent"], target_keys=s["target_keys"], target_values=s["target_values"])
    return [kept, lengths, weights, s["target_keys"], s["target_values"]]


def run(state):
    op = state["case"]["op"]
    if own:
        return {"paged": _own_paged, "window": _own_window, "append": _own_append, "evict": _own_evict}[op](state)
    return {"paged": _plain_paged, "window": _plain_window, "append": _plain_append, "evict": _plain_evict}[op](state)


# ---- what a pass cannot do without --------------------------------------------------------------------------------
def _visible(n, window, sinks):
    """How many of n cache rows the newest token sees."""
    if not window or n <= window:
        return n
    return min(n, window + min(sinks, n - window))


def work(case):
    size, kv, dim = _BYTES[case["type"]], case["kv_heads"], case["dim"]
    row = kv * dim * size
    if case["op"] == "window":
        new, earlier = _prompt(case)
        pairs = sum(_visible(e + i + 1, case["window"], case["sinks"]) for n, e in zip(new, earlier) for i in range(n))
        rows = sum(new)
        return {"bytes": 2 * rows * case["heads"] * dim * size + 2 * (rows + sum(earlier)) * row,
                "flops": 4.0 * pairs * case["heads"] * dim}
    lengths = _lengths(case)
    if case["op"] == "paged":
        seen = sum(_visible(n, case["window"], case["sinks"]) for n in lengths)
        total = 2 * seen * row + 2 * case["batch"] * case["heads"] * dim * size
        return {"bytes": total + (8 * seen * kv if case["weights"] else 0), "flops": 4.0 * seen * case["heads"] * dim}
    if case["op"] == "append":
        return {"bytes": 4 * sum(_appended(case, lengths)) * row, "flops": 0}
    kept = sum(min(n, case["budget"]) for n in lengths)
    return {"bytes": 4 * kept * row + 4 * kv * (sum(lengths) + 2 * kept), "flops": 0}


# ---- the same in 64 bits, sequence by sequence --------------------------------------------------------------------
def _attend64(q, k, v, first, window, sinks):
    """q [n, heads, d] at positions first .., over k, v [m, kv_heads, d]: outputs and weights per head, one head at a time."""
    n, h, d = q.shape
    m, kv = k.shape[:2]
    out, spent = torch.zeros(n, h, d, dtype=torch.float64, device=q.device), []
    far = torch.arange(first, first + n, device=q.device)[:, None] - torch.arange(m, device=q.device)[None, :]
    hidden = far < 0
    if window:
        hidden |= (far >= window) & (torch.arange(m, device=q.device)[None, :] >= sinks)
    for head in range(h):
        e = (q[:, head].double() @ k[:, head * kv // h].double().T) * d ** -0.5
        e = torch.where(hidden, torch.full_like(e, -1e300), e)
        e = torch.where(hidden, torch.zeros_like(e), torch.exp(e - e.max(dim=1).values[:, None]))
        e = e / e.sum(1, keepdim=True).clamp_min(1e-300)
        out[:, head] = e @ v[:, head * kv // h].double()
        spent.append(e if n == 1 else None)
    return out, spent


def _rows64(pages, table_row, n):
    return torch.cat([pages[i] for i in table_row.tolist() if i >= 0])[:n] if n else pages[0][:0]


def exact(case, seed):
    s = prepare(case, seed)
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    if case["op"] == "window":
        qo, ko, parts = s["query_offsets"].tolist(), s["key_offsets"].tolist(), []
        for a, b, c, d in zip(qo, qo[1:], ko, ko[1:]):
            parts.append(_attend64(s["query"][a:b], s["keys"][c:d], s["values"][c:d], (d - c) - (b - a), window, sinks)[0])
        return [torch.cat(parts)]
    lengths, table = s["lengths"].tolist(), s["table"]
    if case["op"] == "paged":
        outs, totals = [], torch.zeros(case["batch"], case["kv_heads"], table.shape[1] * case["page"],
                                       dtype=torch.float64, device="cuda")
        for b, n in enumerate(lengths):
            k, v = (_rows64(s[x], table[b], n) for x in ("key_pages", "value_pages"))
            out, spent = _attend64(s["query"][b:b + 1], k, v, n - 1, window, sinks)
            outs.append(out)
            for head, w in enumerate(spent):
                totals[b, head * case["kv_heads"] // len(spent), :n] += w[0]
        return [torch.cat(outs)] + ([totals] if case["weights"] else [])
    if case["op"] == "append":
        counts, at = _appended(case, lengths), 0
        for b, (n, c) in enumerate(zip(lengths, counts)):
            ids = table[b].tolist()
            for lo in range((n - c) // case["page"], -(-n // case["page"])):
                first, last = max(lo * case["page"], n - c), min((lo + 1) * case["page"], n)
                src = slice(at + first - (n - c), at + last - (n - c))
                dst = slice(first - lo * case["page"], last - lo * case["page"])
                s["key_pages"][ids[lo], dst] = s["keys"][src]
                s["value_pages"][ids[lo], dst] = s["values"][src]
            at += c
        return [s["key_pages"].double(), s["value_pages"].double()]
    page, kv, width = case["page"], case["kv_heads"], s["target"].shape[1] * case["page"]
    kept_all = torch.full((case["batch"], kv, case["budget"]), -1, dtype=torch.int32, device="cuda")
    weights = torch.zeros(case["batch"], kv, width, dtype=torch.float64, device="cuda")
    pools = [s["target_keys"].double(), s["target_values"].double()]
    for b, n in enumerate(lengths):
        rows = [_rows64(s[x], table[b], n) for x in ("key_pages", "value_pages")]
        for head in range(kv):
            w = s["weights"][b, head, :n].double().cpu().numpy()
            last = max(n - case["recent"], min(case["sinks"], n))
            middle = sorted(range(min(case["sinks"], n), last), key=lambda t: (-w[t], t))
            fixed = list(range(min(case["sinks"], n))) + list(range(last, n))
            rest = max(0, min(n, case["budget"]) - len(fixed))
            keep = torch.tensor(sorted(fixed + middle[:rest]), device="cuda")
            m = len(keep)
            kept_all[b, head, :m] = keep
            weights[b, head, :m] = s["weights"][b, head][keep].double()
            t = torch.arange(m, device="cuda")
            ids = s["target"][b][t // page].long()
            for pool, r in zip(pools, rows):
                pool[ids, t % page, head] = r[keep, head].double()
    return [kept_all, torch.tensor([min(n, case["budget"]) for n in lengths], dtype=torch.int32, device="cuda"), weights,
            *pools]
