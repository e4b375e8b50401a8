"""Measured cases of the operators for batches that continue one shared prefix.

A long prefix (a system prompt, an image, a video) is prefilled once: its rows
are rotated with positions of one or several axes and appended to the paged
cache.  Many sequences then continue it; each holds only its own tokens and
attends the prefix and itself.  Three operators:

* ``rope_axes``: rotate q and k rows by a table, each pair of dims by the
  position of its axis;
* ``append_rotary``: rotate q and k, store k and v at the rows' slots of the
  paged pool;
* ``shared_prefix``: attention of a decode, verify or prompt-extension block
  over the shared prefix and each sequence's own pages.

``run`` is the plain form in elementary torch operations, or, with ``own``
true, the framework's calls; ``exact`` restates the definitions in 64 bits.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
_BS = 16  # tokens per page, the framework's default

# (q heads, kv heads, head_dim): the repository's 1.5B, 0.5B and 3B target and
# draft shapes, a generic wide-group and a multi-head shape
_HEADS = [(12, 2, 128), (14, 2, 64), (16, 2, 128), (32, 8, 128), (8, 8, 64)]
_SECTIONS = {128: "16,24,24", 64: "8,12,12"}


def _engine():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "speculative-decoding-lab_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import engine
    from engine import layer_ops

    return engine, layer_ops


# ------------------------------------------------------------------- cases
def _rope(name, tokens, heads, dtype, sections, reach, rotary=0):
    return {"name": name, "op": "rope_axes", "tokens": tokens, "hq": heads[0], "hkv": heads[1], "d": heads[2],
            "dtype": dtype, "sections": sections, "reach": reach, "rotary": rotary or heads[2]}


def _append(name, seqs, new, heads, dtype, sections, reach, padded, lens):
    return {"name": name, "op": "append_rotary", "seqs": seqs, "new": new, "hq": heads[0], "hkv": heads[1],
            "d": heads[2], "dtype": dtype, "sections": sections, "reach": reach, "padded": padded, "lens": lens}


def _prefix(name, batch, chunk, prefix, lo, hi, heads, dtype, lens):
    return {"name": name, "op": "shared_prefix", "batch": batch, "chunk": chunk, "prefix": prefix, "own_lo": lo,
            "own_hi": hi, "hq": heads[0], "hkv": heads[1], "d": heads[2], "dtype": dtype, "lens": lens}


def listed():
    return [
        # one image of 37 x 37 patches between text
        _rope("rope image", 1369, (12, 2, 128), "bf16", "16,24,24", 4096),
        # a video prompt of 32 frames of 25 x 25 patches and some text, the wide-group shape
        _rope("rope video", 20250, (32, 8, 128), "bf16", "16,24,24", 32768),
        # the verify block of a small fp32 run, rotating half of each head
        _rope("rope verify fp32", 23, (8, 8, 64), "fp32", "", 2048, 32),
        # one sequence's decode step: launch latency
        _append("append decode 1", 1, 1, (12, 2, 128), "bf16", "", 4096, 0, 1),
        # a draft decode step of a padded serving batch
        _append("append decode 224", 224, 1, (14, 2, 64), "fp16", "", 8192, 1, 2),
        # a chunked prefill: 18 rows of prompts, the last ones padded, three axes
        _append("append prefill", 18, 997, (12, 2, 128), "bf16", "16,24,24", 32768, 1, 3),
        # the smallest call: two continuations of a short prompt
        _prefix("attend decode 2", 2, 1, 529, 1, 40, (12, 2, 128), "bf16", 4),
        # decode of a serving batch under a long system prompt
        _prefix("attend decode 64", 64, 1, 8192, 1, 1024, (12, 2, 128), "bf16", 5),
        # draft-model decode, a large batch
        _prefix("attend decode 256 d64", 256, 1, 2051, 1, 700, (14, 2, 64), "fp16", 6),
        # the verify block of five drafts
        _prefix("attend verify 32", 32, 6, 4001, 1, 512, (12, 2, 128), "bf16", 7),
        # questions of 96 tokens about one long document
        _prefix("attend extend 16", 16, 96, 6000, 0, 64, (16, 2, 128), "bf16", 8),
        # the largest: the verify block of a full batch under a very long prefix
        _prefix("attend verify 256", 256, 6, 16384, 64, 1024, (12, 2, 128), "bf16", 9),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope_axes", "append_rotary", "shared_prefix", "shared_prefix", "shared_prefix"])
    heads = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    sections = rng.choice(["", _SECTIONS[heads[2]]])
    reach = _log(rng, 1024, 32768)
    if kind == "rope_axes":
        rotary = rng.choice([heads[2], heads[2] // 2]) if not sections else heads[2]
        c = _rope("", _log(rng, 1, 20000), heads, dtype, sections, reach, rotary)
    elif kind == "append_rotary":
        new = rng.choice([1, rng.randint(2, 9), _log(rng, 16, 1024)])
        seqs = _log(rng, 1, max(1, min(512, 16384 // new)))
        c = _append("", seqs, new, heads, dtype, sections, reach, rng.randint(0, 1), rng.randint(0, 999))
    else:
        if dtype == "fp32":  # the small fp32 shapes of the parity runs
            heads = rng.choice([(4, 2, 64), (4, 2, 16)])
        chunk = rng.choice([1, 1, rng.randint(2, 9), _log(rng, 10, 200)])
        # rows x prefix bounded by the largest listed case's
        batch = _log(rng, 1, max(1, min(512, 4096 // chunk)))
        most = 256 * 6 * 12 * 128 * 16384 // (batch * chunk * heads[0] * heads[2])
        prefix = _log(rng, 1, max(2, min(32768 if dtype != "fp32" else 4096, most // 2)))
        lo = rng.choice([0, 1, 16])
        hi = lo + _log(rng, 1, max(2, min(2048, 262144 // batch)))
        c = _prefix("", batch, chunk, prefix, lo, hi, heads, dtype, rng.randint(0, 999))
    del c["name"]
    return c


# ------------------------------------------------------------------ layout
def _starts(case):
    """Own tokens of each sequence before the block (attention), or already cached (append)."""
    r = random.Random(case["lens"])
    if case["op"] == "append_rotary":
        return [r.randint(0, 40) for _ in range(case["seqs"])]
    return [r.randint(case["own_lo"], case["own_hi"]) for _ in range(case["batch"])]


def _counts(case):
    """New rows of each sequence of an append: padded batches have a ragged tail."""
    r = random.Random(case["lens"] + 1)
    return [max(1, case["new"] - r.randint(0, case["new"] // 3)) if case["padded"] else case["new"]
            for _ in range(case["seqs"])]


def _reserves(case):
    """The cache's reserve calls, in order: (sequences, starts, counts).  Members grow in three interleaved
    pieces, so their pages scatter."""
    starts = _starts(case)
    n = len(starts)
    if case["op"] == "append_rotary":
        return [(list(range(n)), [0] * n, starts), (list(range(n)), starts, _counts(case))]
    calls = [([0], [0], [case["prefix"]])]
    done = [0] * n
    for piece in range(3):
        upto = [s + case["chunk"] if piece == 2 else (s + case["chunk"]) * (piece + 1) // 3 for s in starts]
        calls.append((list(range(1, n + 1)), list(done), [u - x for u, x in zip(upto, done)]))
        done = upto
    return calls


def _tables(case):
    """Page tables as the cache's allocator hands pages out: from the last page of the pool down."""
    calls = _reserves(case)
    need = {}
    for sids, starts, counts in calls:
        for sid, s, c in zip(sids, starts, counts):
            if c > 0:
                need[sid] = max(need.get(sid, 0), -(-(s + c) // _BS))
            need.setdefault(sid, 0)
    cap = sum(need.values()) + 2
    tables, top = {sid: [] for sid in need}, cap
    for sids, starts, counts in calls:
        for sid, s, c in zip(sids, starts, counts):
            while c > 0 and len(tables[sid]) < -(-(s + c) // _BS):
                top -= 1
                tables[sid].append(top)
    return tables, cap


def _sections(case):
    return [int(s) for s in case["sections"].split(",")] if case["sections"] else None


def _table(reach, rotary, dev):
    """cos / sin of every position, (reach, 2, rotary) fp32: angles in 64 bits, as the far ones need."""
    inv = 1e6 ** (-torch.arange(0, rotary, 2, dtype=torch.float64, device=dev) / rotary)
    ang = torch.arange(reach, dtype=torch.float64, device=dev)[:, None] * inv
    ang = torch.cat((ang, ang), -1)
    return torch.stack((ang.cos(), ang.sin()), 1).float().contiguous()


def _cache(case, tables, cap, members, dev):
    """The framework's cache with the case's pages reserved; the last reserve's slots."""
    engine, _ = _engine()
    kv = engine.PagedKVCache(1, case["hkv"], case["d"], cap, _BS, dev, _DTYPES[case["dtype"]], max_seqs=members)
    for sid in range(members):
        kv.add_sequence(sid)
    slots = None
    for call in _reserves(case):
        slots = kv.reserve(*call)
    return kv, slots


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = _DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dt)

    s = {"op": case["op"], "case": dict(case)}
    if case["op"] == "shared_prefix":
        n, chunk = case["batch"], case["chunk"]
        tables, cap = _tables(case)
        # queries somewhat longer than keys: peaked rows, as trained heads have
        s["q"] = normal(n, chunk, hq, d) * 2
        k, v = normal(cap * _BS, hkv, d), normal(cap * _BS, hkv, d)
        starts = _starts(case)
        if own:
            engine, _ = _engine()
            kv, _slots = _cache(case, tables, cap, n + 1, dev)
            kv.append(0, torch.arange(cap * _BS, dtype=torch.int32, device=dev), k, v)
            s["kv"] = kv
            s["batch"] = engine.SharedPrefixBatch.from_lists(kv, 0, case["prefix"], list(range(1, n + 1)), starts, chunk)
        else:
            s["k"], s["v"] = k, v
            width = max(len(tables[b]) for b in range(1, n + 1))
            s["prefix_pages"] = torch.tensor(tables[0], device=dev)
            s["pages"] = torch.tensor([tables[b] + [0] * (width - len(tables[b])) for b in range(1, n + 1)], device=dev)
            s["starts"] = torch.tensor(starts, device=dev)
        return s
    rotary = case.get("rotary", d)
    s["table"] = _table(case["reach"], rotary, dev)
    sections = _sections(case)
    axes = len(sections) if sections else 1
    tokens = case["tokens"] if case["op"] == "rope_axes" else case["seqs"] * case["new"]
    # q, k and v are column blocks of one projection's rows
    qkv = normal(tokens, (hq + 2 * hkv) * d)
    s["q"] = qkv[:, :hq * d].view(tokens, hq, d)
    s["k"] = qkv[:, hq * d:(hq + hkv) * d].view(tokens, hkv, d)
    s["v"] = qkv[:, (hq + hkv) * d:].view(tokens, hkv, d)
    # rows run along a prompt, or over frames of 25 x 25 patches, from a random base
    base = torch.randint(0, max(1, case["reach"] // 2), (axes, 1), generator=g, device=dev)
    t = torch.arange(tokens, device=dev)
    grid = torch.stack((t // 625, t // 25 % 25, t % 25)) if axes == 3 else t[None]
    s["positions"] = (base + grid) % case["reach"]
    s["sections"] = sections
    if axes == 1:
        s["positions"] = s["positions"][0].contiguous()
    if case["op"] == "append_rotary":
        tables, cap = _tables(case)
        seqs, new = case["seqs"], case["new"]
        starts, counts = _starts(case), _counts(case)
        if own:
            kv, flat = _cache(case, tables, cap, seqs, dev)
            s["kv"] = kv
            grid = torch.full((seqs * new,), -1, dtype=torch.int32, device=dev)
            live = torch.tensor([b * new + j for b in range(seqs) for j in range(counts[b])], device=dev)
            grid[live] = flat
            s["slots"] = grid
        else:
            slots = [tables[b][(starts[b] + j) // _BS] * _BS + (starts[b] + j) % _BS if j < counts[b] else -1
                     for b in range(seqs) for j in range(new)]
            s["slots"] = torch.tensor(slots, dtype=torch.int32, device=dev)
            # one spare row takes what padding rows would store
            s["k_pool"] = torch.zeros((cap * _BS + 1, hkv, d), dtype=dt, device=dev)
            s["v_pool"] = torch.zeros((cap * _BS + 1, hkv, d), dtype=dt, device=dev)
    return s


# --------------------------------------------------------------- plain forms
def _angles(s):
    """cos and sin of each row and pair of dims, (tokens, 1, rotary / 2)."""
    pos = s["positions"].reshape(-1, s["positions"].shape[-1])
    half = s["table"].shape[-1] // 2
    if s["sections"]:
        axis = torch.arange(len(s["sections"]), device=pos.device).repeat_interleave(
            torch.tensor(s["sections"], device=pos.device), output_size=half)
    else:
        axis = torch.zeros(half, dtype=torch.long, device=pos.device)
    pick = pos.t()[:, axis]  # (tokens, half): the position that turns each pair
    pair = torch.arange(half, device=pos.device)
    return s["table"][pick, 0, pair][:, None, :], s["table"][pick, 1, pair][:, None, :]


def _turn(x, cos, sin):
    half = cos.shape[-1]
    f = x.float()
    a, b, rest = f[..., :half], f[..., half:2 * half], f[..., 2 * half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin, rest), -1).to(x.dtype)


def _attend(s):
    """Logits of every row over the prefix and over its own pages, one softmax over both."""
    q = s["q"].float()
    n, chunk, hq, d = q.shape
    prefix, hkv = s["case"]["prefix"], s["case"]["hkv"]
    k, v = s["k"].view(-1, _BS, hkv, d), s["v"].view(-1, _BS, hkv, d)
    kp = k[s["prefix_pages"]].reshape(-1, hkv, d)[:prefix].float().permute(1, 2, 0)  # (hkv, d, P)
    vp = v[s["prefix_pages"]].reshape(-1, hkv, d)[:prefix].float().permute(1, 0, 2)
    ko = k[s["pages"]].reshape(n, -1, hkv, d).float().permute(0, 2, 3, 1)  # (n, hkv, d, L)
    vo = v[s["pages"]].reshape(n, -1, hkv, d).float().permute(0, 2, 1, 3)
    span = ko.shape[-1]
    g = hq // hkv
    qg = q.view(n, chunk, hkv, g, d) / math.sqrt(d)
    qp = qg.permute(2, 0, 1, 3, 4).reshape(hkv, n * chunk * g, d)
    qo = qg.permute(0, 2, 1, 3, 4).reshape(n, hkv, chunk * g, d)
    sp = torch.matmul(qp, kp).view(hkv, n, chunk, g, prefix)
    so = torch.matmul(qo, ko).view(n, hkv, chunk, g, span)
    limit = s["starts"][:, None] + torch.arange(chunk, device=q.device)  # last own key of row (b, j)
    hidden = torch.arange(span, device=q.device) > limit[..., None]  # (n, chunk, L)
    so = so.masked_fill_(hidden[:, None, :, None, :], float("-inf"))
    top = torch.maximum(sp.amax(-1), so.amax(-1).permute(1, 0, 2, 3))  # (hkv, n, chunk, g)
    sp = sp.sub_(top[..., None]).exp_()
    so = so.sub_(top.permute(1, 0, 2, 3)[..., None]).exp_()
    total = sp.sum(-1) + so.sum(-1).permute(1, 0, 2, 3)
    out = torch.matmul(sp.view(hkv, n * chunk * g, prefix), vp).view(hkv, n, chunk, g, d)
    out = out + torch.matmul(so.view(n, hkv, chunk * g, span), vo).view(n, hkv, chunk, g, d).permute(1, 0, 2, 3, 4)
    out = out / total[..., None]
    return out.permute(1, 2, 0, 3, 4).reshape(n, chunk, hq, d).to(s["q"].dtype)


def run(s):
    if own:
        engine, layer_ops = _engine()
        if s["op"] == "rope_axes":
            return layer_ops.rope_axes(s["q"], s["k"], s["table"], s["positions"], s["sections"])
        if s["op"] == "append_rotary":
            kv = s["kv"]
            q = kv.append_rotary(0, s["slots"], s["k"], s["v"], s["table"], s["positions"], s["sections"], query=s["q"])
            return q, kv._k[0].view(-1, kv.num_kv_heads, kv.head_dim), kv._v[0].view(-1, kv.num_kv_heads, kv.head_dim)
        return engine.paged_attention_shared_prefix(s["q"], s["kv"], 0, s["batch"])
    if s["op"] == "shared_prefix":
        return _attend(s)
    cos, sin = _angles(s)
    q, k = _turn(s["q"], cos, sin), _turn(s["k"], cos, sin)
    if s["op"] == "rope_axes":
        return q, k
    slots = s["slots"].long()
    at = torch.where(slots < 0, s["k_pool"].shape[0] - 1, slots)
    s["k_pool"][at] = k
    s["v_pool"][at] = s["v"]
    return q * (slots >= 0)[:, None, None], s["k_pool"][:-1], s["v_pool"][:-1]


# ------------------------------------------------------------------ the work
def work(case):
    size, hq, hkv, d = _SIZE[case["dtype"]], case["hq"], case["hkv"], case["d"]
    if case["op"] == "shared_prefix":
        n, chunk, prefix = case["batch"], case["chunk"], case["prefix"]
        ends = [s + chunk for s in _starts(case)]
        own_pairs = sum(chunk * e - chunk * (chunk - 1) // 2 for e in ends)
        return {"bytes": 2 * n * chunk * hq * d * size + (prefix + sum(ends)) * 2 * hkv * d * size,
                "flops": 4 * d * hq * (n * chunk * prefix + own_pairs)}
    rotary = case.get("rotary", d)
    axes = len(_sections(case)) if case["sections"] else 1
    if case["op"] == "rope_axes":
        rows, heads = case["tokens"], hq + hkv
    else:
        rows, heads = sum(_counts(case)), hq + 2 * hkv
    turned = rows * (hq + hkv) * rotary
    # distinct angle rows are read once: at most one per token, one half of the duplicated columns
    return {"bytes": 2 * rows * heads * d * size + min(rows, case["reach"]) * rotary * 4 + rows * axes * 8,
            "flops": 3 * turned}


# ------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """From the definitions, in 64 bits: complex rotations, and one dense softmax per sequence."""
    s = prepare(case, seed)
    if s["op"] == "shared_prefix":
        hkv, d = case["hkv"], case["d"]
        prefix, chunk, g = case["prefix"], case["chunk"], case["hq"] // case["hkv"]
        k, v = s["k"].double(), s["v"].double()
        tables, _ = _tables(case)
        off = torch.arange(_BS, device=k.device)

        def rows(pages, count):
            at = (torch.tensor(pages, dtype=torch.long, device=k.device)[:, None] * _BS + off).reshape(-1)[:count]
            return k[at], v[at]

        kp, vp = rows(tables[0], prefix)
        out = torch.empty(s["q"].shape, dtype=torch.float64, device=k.device)
        for b, start in enumerate(_starts(case)):
            kb, vb = rows(tables[b + 1], start + chunk)
            keys, vals = torch.cat((kp, kb)), torch.cat((vp, vb))
            place = torch.arange(len(keys), device=k.device)
            for h in range(hkv):
                q = s["q"][b, :, h * g:(h + 1) * g].double()
                w = torch.tensordot(q, keys[:, h], dims=([2], [1])) * d ** -0.5  # (chunk, g, keys)
                last = prefix + start + torch.arange(chunk, device=k.device)
                w[(place[None, :] > last[:, None])[:, None, :].expand_as(w)] = float("-inf")
                w = torch.softmax(w, -1)
                out[b, :, h * g:(h + 1) * g] = torch.tensordot(w, vals[:, h], dims=([2], [0]))
        return out
    table = s["table"].double()
    half = table.shape[-1] // 2
    pos = s["positions"].reshape(-1, s["positions"].shape[-1])
    unit = torch.complex(table[:, 0, :half], table[:, 1, :half])
    parts, first = [], 0
    for a, width in enumerate(s["sections"] or [half]):
        parts.append(unit[pos[a], first:first + width])
        first += width
    unit = torch.cat(parts, 1)[:, None, :]

    def turn(x):
        z = x.double()
        w = torch.complex(z[..., :half].contiguous(), z[..., half:2 * half].contiguous()) * unit
        return torch.cat((w.real, w.imag, z[..., 2 * half:]), -1)

    if s["op"] == "rope_axes":
        return turn(s["q"]), turn(s["k"])
    live = torch.nonzero(s["slots"] >= 0).reshape(-1)
    at = s["slots"][live].long()
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device=table.device)
    q[live] = turn(s["q"])[live]
    k_pool = s["k_pool"][:-1].double()
    v_pool = s["v_pool"][:-1].double()
    k_pool[at] = turn(s["k"])[live]
    v_pool[at] = s["v"][live].double()
    return q, k_pool, v_pool
