"""Operators of serving with an 8-bit cache, rotary positions, beams and a pool of pages, as
measurable cases.

A server that holds several requests' sequences in one pool of pages needs, around a model's
matrices: queries and keys rotated by their positions, new keys and values written to pages of
8 bits, attention over such pages, the best continuations of every request's beams, and the
pages of sequences forked as the beams go on, and moved together when the pool is fragmented.
Head shapes and vocabularies are those of the package's model presets.
"""
import math
import random

import torch

own = False
GPU = "cuda:0"

# query heads, KV heads, head size, vocabulary
MODELS = {
    "smollm2-360m": (15, 5, 64, 49152),
    "qwen2.5-0.5b": (14, 2, 64, 151936),
    "llama-3.2-1b": (32, 8, 64, 128256),
    "llama-3.1-8b": (32, 8, 128, 128256),
    "qwen3-30b-a3b": (32, 4, 128, 151936),
    "gemma-3-1b": (4, 1, 256, 262144),
}
WINDOW = 512  # gemma-3-1b's window layers
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SMALLEST = 2.0 ** -60  # a block's values that would have a smaller scale count as zeros


def listed():
    def append(name, model, seqs, new, length, page, block, src):
        return {"name": name, "op": "append", "model": model, "seqs": seqs, "new": new, "chunks": seqs, "len": length, "page": page, "block": block, "src": src}

    def attend(name, model, seqs, new, chunks, length, page, block, ty, window=0):
        return {"name": name, "op": "attend", "model": model, "seqs": seqs, "new": new, "chunks": chunks, "len": length, "page": page, "block": block,
                "type": ty, "window": window}

    def rotary(name, model, rows, dims, layout, scaling, src, ty):
        return {"name": name, "op": "rotary", "model": model, "rows": rows, "dims": dims, "layout": layout, "scaling": scaling, "src": src, "type": ty}

    def beam(name, model, requests, beams, keep, ty):
        return {"name": name, "op": "beam", "model": model, "requests": requests, "beams": beams, "keep": keep, "type": ty}

    def pages(name, op, model, seqs, beams, length, page, layers):
        return {"name": name, "op": op, "model": model, "seqs": seqs, "beams": beams, "len": length, "page": page, "layers": layers}

    return [
        # one decode step of 61 sequences into 8-bit pages: most tokens join a block that holds others
        append("append8-tokens-qwen3-30b-a3b", "qwen3-30b-a3b", 61, 1, 3000, 16, 16, "bf16"),
        # the prompts of a few new requests, from the f32 rows that the matrices give
        append("append8-prompts-llama-3.1-8b", "llama-3.1-8b", 7, 1500, 1500, 64, 32, "f32"),
        # the smallest call: a few short chats with a small model, 15 heads on 5
        attend("token8-smollm2-360m-3x190", "smollm2-360m", 3, 1, 0, 190, 16, 16, "f16"),
        # one decode step of a busy server, ragged lengths
        attend("token8-llama-3.1-8b-48x4000", "llama-3.1-8b", 48, 1, 0, 4000, 16, 16, "f16"),
        # the next token of one very long document
        attend("token8-qwen3-30b-a3b-1x100003", "qwen3-30b-a3b", 1, 1, 0, 100003, 64, 32, "bf16"),
        # a long prompt's chunks beside other sequences' single tokens in one batch
        attend("chunk8-llama-3.1-8b-13x8200", "llama-3.1-8b", 13, 509, 3, 8200, 32, 16, "bf16"),
        # one decode step's queries and keys, halves, the whole head
        rotary("rotary-tokens-qwen2.5-0.5b-61", "qwen2.5-0.5b", 61, 64, "halves", "none", "f16", "f16"),
        # packed prompts of a long-context model: part of the head, interleaved pairs, frequencies scaled by parts
        rotary("rotary-prompts-llama-3.1-8b-9001", "llama-3.1-8b", 9001, 96, "pairs", "parts", "f32", "bf16"),
        # one step of one request with 4 beams
        beam("beam-qwen3-30b-a3b-1x4", "qwen3-30b-a3b", 1, 4, 4, "f32"),
        # a batch of requests with 8 beams, twice as many candidates kept for those that may end
        beam("beam-llama-3.1-8b-24x8", "llama-3.1-8b", 24, 8, 16, "bf16"),
        # the beams' caches after such a step: rows reordered, shared pages, copies of partial ones
        pages("fork-llama-3.1-8b-24x8", "fork", "llama-3.1-8b", 192, 8, 700, 16, 4),
        # a pool that long sequences have left full of holes
        pages("compact-qwen3-30b-a3b-40x3000", "compact", "qwen3-30b-a3b", 40, 1, 3000, 32, 6),
    ]


def draw(rng):
    def log(lo, hi):
        return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    most = max(_size(c) for c in listed())
    while True:
        op = rng.choice(["append", "attend", "attend", "attend", "rotary", "rotary", "beam", "beam", "fork", "compact"])
        model = rng.choice(sorted(MODELS))
        H, KV, hd, V = MODELS[model]
        ty = rng.choice(["f16", "bf16"])
        page = rng.choice([16, 32, 64, 128])
        block = rng.choice([b for b in (16, 32, 64) if b <= page])
        if op == "append":
            new = rng.choice([1, log(2, 1500)])
            seqs = log(1, 100)
            c = {"op": op, "model": model, "seqs": seqs, "new": new, "chunks": seqs, "len": max(new, log(1, 4000)), "page": page, "block": block,
                 "src": rng.choice(["f32", "f16", "bf16"])}
            good = seqs * new <= 20000
        elif op == "attend":
            new = rng.choice([1, 1, log(2, 8), log(9, 600)])
            seqs = log(1, 100)
            c = {"op": op, "model": model, "seqs": seqs, "new": new, "chunks": rng.randint(1, seqs) if new > 1 else 0,
                 "len": max(new, log(16, 100000)), "page": page, "block": block, "type": ty,
                 "window": WINDOW if model == "gemma-3-1b" and rng.random() < 0.5 else 0}
            good = seqs * c["len"] <= 200000 and seqs * new * c["len"] * H <= 2.5e9
        elif op == "rotary":
            c = {"op": op, "model": model, "rows": log(1, 12000), "dims": rng.choice([hd, hd, hd // 2, hd // 4 * 3]), "layout": rng.choice(["halves", "pairs"]),
                 "scaling": rng.choice(["none", "linear", "parts"]), "src": rng.choice(["f32", ty]), "type": ty}
            good = c["rows"] * (H + KV) * hd <= 5e7
        elif op == "beam":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 16])
            c = {"op": op, "model": model, "requests": log(1, 60), "beams": beams, "keep": rng.choice([beams, 2 * beams]), "type": rng.choice(["f32", "f16", "bf16"])}
            good = c["requests"] * beams * V <= 4e7
        else:
            beams = rng.choice([2, 4, 5, 8]) if op == "fork" else 1
            c = {"op": op, "model": model, "seqs": beams * log(1, 200 // beams), "beams": beams, "len": log(16, 4000), "page": page, "layers": rng.randint(1, 6)}
            good = c["seqs"] * (c["len"] + page) * KV * hd * 4 * c["layers"] <= 3e9
        if good and _size(c) <= most:
            return c


def _size(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _lengths(case):
    """(new tokens, length with them) of every sequence; lengths from a tenth of the longest up, and the longest first"""
    r = random.Random(case["seqs"] * 1000003 + case["len"])
    n = case["seqs"]
    if case["op"] == "fork":  # the beams of a request are of one length
        each = [max(1, round(case["len"] * 10 ** -r.random())) for _ in range(n // case["beams"])]
        return [(1, x) for x in each for _ in range(case["beams"])]
    lens = [case["len"]] + [max(1, round(case["len"] * 10 ** -r.random())) for _ in range(n - 1)]
    if case["op"] == "append":  # every sequence brings about as much as the longest
        return [(min(x, max(1, round(case["new"] * r.uniform(0.5, 1.0)))) if case["new"] > 1 else 1, x) for x in lens]
    if case["op"] == "compact":
        return [(1, x) for x in lens]
    return [(min(case["new"], x) if i < case["chunks"] else 1, x) for i, x in enumerate(lens)]


def _pairs(new, length, window):
    """query and position pairs that one head computes"""
    seen = range(length - new + 1, length + 1)
    return sum(min(p, window) for p in seen) if window else new * (seen[0] + seen[-1]) // 2


def _read(new, length, window):
    """positions that at least one new token sees"""
    return min(length, window + new - 1) if window else length


def _parents(case):
    """the row that each row goes on from: a third of a request's beams carry on two or three of its rows"""
    r = random.Random(case["seqs"] * 31 + case["len"])
    W = case["beams"]
    return [a + min(r.randrange(W), r.randrange(W)) for a in range(0, case["seqs"], W) for _ in range(W)]


def _pool(case):
    """pages of every sequence, and of the pool"""
    held = [-(-x // case["page"]) for _, x in _lengths(case)]
    return held, sum(held) * 3 // 2 + case["seqs"] + 3 if case["op"] == "compact" else sum(held) + case["seqs"] + 3


def _moved(case):
    """pages that a fork copies or a compaction moves"""
    held, n_pages = _pool(case)
    if case["op"] == "fork":
        src = _parents(case)
        return sum(case["beams"] and x % case["page"] > 0 for i, (_, x) in enumerate(_lengths(case)) if src[i] in src[:i] or (src[i] != i and src[src[i]] == src[i]))
    return sum(p >= sum(held) for p in _places(case))


def _places(case):
    """page ids in the order in which sequences take them"""
    held, n_pages = _pool(case)
    order = list(range(n_pages))
    random.Random(case["seqs"] + 7 * case["len"]).shuffle(order)
    return order[:sum(held)]


def work(case):
    H, KV, hd, V = MODELS[case["model"]]
    if case["op"] == "rotary":
        n = case["rows"] * (H + KV) * hd
        return {"bytes": n * (TYPES[case["src"]].itemsize + TYPES[case["type"]].itemsize) + 4 * case["rows"], "flops": 3 * n * case["dims"] // hd}
    if case["op"] == "beam":
        n = case["requests"] * case["beams"] * V
        return {"bytes": n * TYPES[case["type"]].itemsize + case["requests"] * (8 * case["beams"] + 12 * case["keep"]), "flops": 4 * n}
    if case["op"] in ("fork", "compact"):
        held, n_pages = _pool(case)
        return {"bytes": _moved(case) * 2 * KV * hd * case["page"] * 2 * 2 * case["layers"] + 8 * sum(held) + 8 * n_pages, "flops": 0}
    lens = _lengths(case)
    rows = sum(n for n, _ in lens)
    if case["op"] == "append":
        return {"bytes": 2 * rows * KV * hd * (TYPES[case["src"]].itemsize + 1) + 8 * (rows // case["block"] + len(lens)) * KV + 8 * rows, "flops": 0}
    positions = sum(_read(n, x, case["window"]) for n, x in lens)
    pairs = sum(_pairs(n, x, case["window"]) for n, x in lens)
    return {"bytes": 4 * rows * H * hd + 2 * positions * KV * hd + 8 * positions // case["block"] * KV, "flops": 4 * hd * H * pairs}


def _frequencies(dims, scaling, base=500000.0, factor=8.0, original=8192):
    """angles per position, f64, and what the rotated values are multiplied by"""
    f = base ** (-2 * torch.arange(dims // 2, dtype=torch.float64) / dims)
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "parts":  # fast ones as they are, slow ones stretched, a ramp between 32 turns and 1 of the original context
        def at(turns):
            return dims * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), dims - 1)
        ramp = ((torch.arange(dims // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        return f / factor * ramp + f * (1 - ramp), 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    H, KV, hd, V = MODELS[case["model"]]
    op = case["op"]
    s = {"case": case}
    if op == "rotary":
        # slices of the fused projection's rows; positions of tokens anywhere in a long context
        qkv = torch.randn(case["rows"], H + 2 * KV, hd, device=GPU, generator=g).to(TYPES[case["src"]])
        s["q"], s["k"] = qkv[:, :H], qkv[:, H:H + KV]
        s["positions"] = torch.randint(0, 131072, (case["rows"],), device=GPU, generator=g, dtype=torch.int32)
        f, s["magnitude"] = _frequencies(case["dims"], case["scaling"])
        s["frequencies"] = f.to(GPU)
        s["q_out"], s["k_out"] = (torch.empty(case["rows"], n, hd, device=GPU, dtype=TYPES[case["type"]]) for n in (H, KV))
    elif op == "beam":
        # logits of a trained model: a wide body, and a few tokens that stand out
        n, W, K = case["requests"], case["beams"], case["keep"]
        x = torch.randn(n * W, V, device=GPU, generator=g) * 2.5 - 3
        at = torch.arange(40, device=GPU) * (V // 40) + torch.randint(0, V // 40, (n * W, 40), device=GPU, generator=g)
        x.scatter_(1, at, torch.rand(n * W, 40, device=GPU, generator=g) * 12 + 4)
        s["logits"] = x.to(TYPES[case["type"]])
        # beams of similar sums, the best first; now and then one that has ended
        s["scores"] = -20 - torch.rand(n, W, device=GPU, generator=g).mul(4).cumsum(1)
        s["finished"] = (torch.rand(n, W, device=GPU, generator=g) < 0.05).int()
        s["next"] = torch.empty(n, K, device=GPU)
        s["parents"], s["tokens"] = (torch.empty(n, K, device=GPU, dtype=torch.int32) for _ in range(2))
    elif op in ("fork", "compact"):
        held, n_pages = _pool(case)
        n, per = len(held), max(held) + 2
        table = torch.full((n, per), -1, dtype=torch.int32)
        places = torch.tensor(_places(case), dtype=torch.int32)
        table[torch.arange(per)[None] < torch.tensor(held)[:, None]] = places
        refs = torch.zeros(n_pages, dtype=torch.int32)
        refs[places.long()] = 1
        # what the host of a server never reads: tables, lengths, pages held, references, and how many pages a call lacked
        lens = torch.tensor([x for _, x in _lengths(case)], dtype=torch.int32)
        s["start"] = torch.cat([table.flatten(), lens, torch.tensor(held, dtype=torch.int32), refs, torch.zeros(2, dtype=torch.int32)]).to(GPU)
        s["state"] = s["start"].clone()
        s["table"], s["lens"], s["held"], s["refs"], s["counts"] = s["state"].split([n * per, n, n, n_pages, 2])
        s["table"] = s["table"].view(n, per)
        s["src"] = torch.tensor(_parents(case), dtype=torch.int32).to(GPU) if op == "fork" else None
        s["caches"] = [torch.randn(n_pages, KV, case["page"], hd, device=GPU, generator=g).to(torch.bfloat16) for _ in range(2 * case["layers"])]
    else:
        lens = _lengths(case)
        new = torch.tensor([n for n, _ in lens])
        s["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).int().to(GPU)
        s["lens"] = torch.tensor([x for _, x in lens], dtype=torch.int32).to(GPU)
        s["max_new"], s["max_len"], s["rows"] = max(n for n, _ in lens), max(x for _, x in lens), int(new.sum())
        page, block = case["page"], case["block"]
        per = -(-s["max_len"] // page)
        need = sum(-(-x // page) for _, x in lens)
        order = torch.randperm(need + 3, device=GPU, generator=g).int()
        used = (torch.arange(per)[None] < -(-s["lens"].cpu()[:, None] // page)).to(GPU)
        table = torch.zeros(len(lens), per, dtype=torch.int32, device=GPU)
        table[used] = order[:need]
        s["table"] = table
        # keys, then values: every KV head's rows of a page lie together; scales of a block and head
        s["codes"] = torch.randint(-127, 128, (2, need + 3, KV, page, hd), device=GPU, generator=g, dtype=torch.int8)
        s["scales"] = torch.rand(2, need + 3, page // block, KV, device=GPU, generator=g) * 0.02 + 0.015
        if op == "append":
            src = torch.randn(s["rows"], 2 * KV, hd, device=GPU, generator=g).to(TYPES[case["src"]])
            s["new_k"], s["new_v"] = src[:, :KV], src[:, KV:]
            # pages that get new tokens, which come back as values
            first = torch.tensor([(x - n) // page for n, x in lens]), torch.tensor([(x - 1) // page for n, x in lens])
            col = torch.arange(per)[None]
            s["written"] = table[((col >= first[0][:, None]) & (col <= first[1][:, None])).to(GPU)].long()
        else:
            s["q"] = (torch.randn(s["rows"], H, hd, device=GPU, generator=g) * 1.5).to(TYPES[case["type"]])
            s["out"] = torch.empty(s["rows"], H, hd, device=GPU, dtype=TYPES[case["type"]])
            s["scale"] = 1 / math.sqrt(hd)
    if own:
        s["call"] = _call(s)
    return s


def _call(s):
    """The framework's call over the state's buffers, which a server makes at every layer or step."""
    from rust_interference_engine_amd import ops

    case = s["case"]
    op = case["op"]
    if op == "rotary":
        return ops.Rotary(s["frequencies"], s["q"], s["k"], s["q_out"], s["k_out"], positions=s["positions"], interleaved=case["layout"] == "pairs",
                          magnitude=s["magnitude"])
    if op == "beam":
        return ops.BeamSelect(s["logits"], s["scores"], s["next"], s["parents"], s["tokens"], finished=s["finished"], pad=2)
    if op in ("fork", "compact"):
        pool = ops.PagePool(s["table"], s["lens"], s["held"], s["refs"], s["counts"], page_size=case["page"])
        return ops.PageFork(pool, s["src"], s["caches"]) if op == "fork" else ops.PageCompact(pool, s["caches"])
    seqs = ops.Seqs(s["starts"], s["lens"], max_new=s["max_new"], max_len=s["max_len"])
    (k, v), (k_scale, v_scale) = s["codes"].transpose(2, 3), s["scales"]
    kv = ops.PagedKv(k, v, s["table"], k_scale=k_scale, v_scale=v_scale)
    if op == "append":
        return ops.PagedAppend(kv, seqs, s["new_k"], s["new_v"])
    return ops.PagedAttention(kv, seqs, s["q"], s["out"], scale=s["scale"], window=case["window"])


def run(s):
    op = s["case"]["op"]
    if op in ("fork", "compact"):  # both change their own input: the pool as it was
        s["state"].copy_(s["start"])
    if own:
        s["call"]()
    else:
        {"append": _append, "attend": _attend, "rotary": _rotary, "beam": _beam, "fork": _fork, "compact": _compact}[op](s)
    if op == "append":
        page, block = s["case"]["page"], s["case"]["block"]
        scale = s["scales"][:, s["written"]]
        return {"values": s["codes"][:, s["written"]].unflatten(3, (page // block, block)) * scale.transpose(2, 3)[..., None, None], "scale": scale}
    return {k: s[k] for k in {"attend": ("out",), "rotary": ("q_out", "k_out"), "beam": ("next", "parents", "tokens"), "fork": ("table", "lens", "held", "refs", "counts", "caches"),
                              "compact": ("table", "refs", "counts", "caches")}[op]}


def _rows(s):
    """sequence and place within its new tokens of every row, and its position in the sequence"""
    starts, r = s["starts"].long(), torch.arange(s["rows"], device=GPU)
    seq = torch.searchsorted(starts, r, right=True) - 1
    at = r - starts[seq]
    return seq, at, (s["lens"].long() - starts[1:] + starts[:-1])[seq] + at


def _append(s):
    page, block = s["case"]["page"], s["case"]["block"]
    codes, scales = s["codes"], s["scales"]
    n_blocks = page // block
    seq, at, pos = _rows(s)
    p, slot = s["table"][seq, pos // page].long(), pos % page
    where = p * n_blocks + slot // block
    x = torch.stack([s["new_k"], s["new_v"]]).float()  # [2, rows, heads, size]
    flat = scales.view(2, -1, scales.shape[3])
    size = torch.zeros_like(flat).index_reduce_(1, where, x.abs().amax(-1), "amax")
    # a block that a sequence's first new token finds begun keeps its scale, or it grows and the codes follow
    start = s["lens"].long() - (s["starts"][1:] - s["starts"][:-1])
    begun = start % block > 0
    p0 = s["table"].gather(1, (start // page).clamp(max=s["table"].shape[1] - 1)[:, None])[:, 0].long()
    b0 = p0 * n_blocks + start % page // block
    was = torch.where(begun[:, None], flat[:, b0], 0.0)
    fresh = (size.double() / 127).float()
    fresh = torch.where(fresh < SMALLEST, 0.0, fresh)
    now = torch.maximum(fresh[:, b0], was)
    fresh[:, b0] = now
    flat[:, where] = fresh[:, where]
    slots = (start % page // block * block)[:, None] + torch.arange(block, device=GPU)
    old = codes[:, p0[:, None], :, slots]  # [sequence, slot, 2, head, size]
    # codes next to a half go by 64 bits
    factor = torch.where(now > 0, was.double() / now.double(), 1.0).permute(1, 0, 2)[:, None, :, :, None]
    again = (old * factor).round().to(torch.int8)
    codes[:, p0[:, None], :, slots] = torch.where((begun[:, None] & (slots < (start % page)[:, None]))[..., None, None, None], again, old)
    scale = fresh[:, where, :, None].double()
    codes[:, p, :, slot] = torch.where(scale > 0, x * (1 / scale), 0.0).round().to(torch.int8).transpose(0, 1)


def _attend(s):
    H, KV, hd, _ = MODELS[s["case"]["model"]]
    block, w = s["case"]["block"], s["case"]["window"]

    def cached(pages, scale):  # [sequence, page, head, slot, size] to [sequence, head, position, size]
        x = pages[s["table"].long()].float() * scale[s["table"].long()].transpose(2, 3).repeat_interleave(block, 3)[..., None]
        return x.transpose(1, 2).flatten(2, 3)

    k, v = cached(s["codes"][0], s["scales"][0]), cached(s["codes"][1], s["scales"][1])
    n, L = k.shape[0], k.shape[2]
    starts, lens = s["starts"].long(), s["lens"].long()
    t = torch.arange(s["max_new"], device=GPU)
    q = s["q"][(starts[:-1, None] + t).clamp(max=s["rows"] - 1)].float() * s["scale"]
    q = q.view(n, -1, KV, H // KV, hd).permute(0, 2, 3, 1, 4).reshape(n, KV, -1, hd)
    pos = (lens - starts[1:] + starts[:-1])[:, None] + t
    j = torch.arange(L, device=GPU)
    hide = j > pos[..., None]
    if w:
        hide |= j <= pos[..., None] - w
    x = torch.matmul(q, k.transpose(2, 3)).view(n, KV, H // KV, -1, L)
    x.masked_fill_(hide[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    x.exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(n, KV, -1, L), v).view(n, KV, H // KV, -1, hd) / total
    seq, at, _ = _rows(s)
    s["out"].copy_(o.permute(0, 3, 1, 2, 4).reshape(n, -1, H, hd)[seq, at])


def _rotary(s):
    dims, pairs = s["case"]["dims"], s["case"]["layout"] == "pairs"
    angle = s["positions"].double()[:, None] * s["frequencies"]  # far positions' angles lose their digits in 32 bits
    cos, sin = (y.float()[:, None] * s["magnitude"] for y in (angle.cos(), angle.sin()))

    def rotated(x, out):
        y = x.float()
        r = y[..., :dims]
        a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :dims // 2], r[..., dims // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        r = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
        out.copy_(torch.cat([r, y[..., dims:]], -1))

    rotated(s["q"], s["q_out"])
    rotated(s["k"], s["k_out"])


def _beam(s):
    x = s["logits"].float()
    n, W, K, V = s["case"]["requests"], s["case"]["beams"], s["case"]["keep"], x.shape[1]
    # a row's best: one whole-number key orders by value, then by index, the lowest first
    bits = (x + 0.0).view(torch.int32).long()
    key = (torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF) << 32) - torch.arange(V, device=GPU)
    ids = (-key.topk(K, -1).values) & 0xFFFFFFFF
    # beams are compared by their sums, which 32 bits would make equal too often
    m = x.amax(-1, keepdim=True).double()
    log_total = (x.double() - m).exp().sum(-1, keepdim=True).log()
    score = s["scores"].double().view(-1, 1) + ((x.gather(1, ids).double() - m) - log_total)
    done = s["finished"].view(-1, 1) != 0
    first = torch.arange(K, device=GPU) == 0
    score = torch.where(done, torch.where(first, s["scores"].double().view(-1, 1), -math.inf), score).view(n, W * K)
    ids = torch.where(done, 2, ids).view(n, W * K)
    best, at = torch.sort(score, stable=True, dim=-1, descending=True)
    at = at[:, :K]
    s["next"].copy_(best[:, :K])
    s["parents"].copy_(at // K + torch.arange(n, device=GPU)[:, None] * W)
    s["tokens"].copy_(ids.gather(1, at))


def _fork(s):
    page, n, cols = s["case"]["page"], *s["table"].shape
    table, lens, held, src, refs = s["table"].clone(), s["lens"].clone().long(), s["held"].clone().long(), s["src"].long(), s["refs"]
    i, n_pages = torch.arange(n, device=GPU), refs.numel()
    children = torch.zeros_like(lens).index_add_(0, src, torch.ones_like(lens))
    # a source's partial page stays with the row itself if it goes on, else with its first child
    heir = torch.full_like(lens, n).index_reduce_(0, src, torch.where(src == i, -1, i), "amin")
    keeps = (heir[src] == i) | (src == i)
    full = lens // page
    need = ~keeps & (lens % page > 0)[src]
    free = refs == 0
    by_rank = torch.full((n_pages + 1,), -1, device=GPU).scatter_(0, torch.where(free, free.cumsum(0) - 1, n_pages), torch.arange(n_pages, device=GPU))
    by_rank[n_pages] = -1
    fresh = by_rank[(need.cumsum(0) - 1).clamp(0, n_pages)]
    c = torch.arange(cols, device=GPU)
    change = torch.where(c < full[:, None], children[:, None] - 1, torch.where(children == 0, -1, 0)[:, None])
    held_pages = c < held[:, None]
    refs.index_add_(0, table.clamp(min=0).long().flatten(), torch.where(held_pages, change, 0).int().flatten())
    new_held = torch.where(keeps, held[src], -(-lens // page)[src])
    rows = torch.where((c == full[src][:, None]) & need[:, None], fresh[:, None], table[src].long())
    s["table"].copy_(torch.where(c < new_held[:, None], rows, -1))
    s["lens"].copy_(lens[src])
    s["held"].copy_(new_held)
    s["counts"][0] = (need & (fresh < 0)).sum()
    at = (need & (fresh >= 0)).nonzero()[:, 0]
    to, of = fresh[at], table[src[at], full[src[at]]].long()
    refs[to] = 1
    for x in s["caches"]:
        x[to] = x[of]


def _compact(s):
    refs, table = s["refs"], s["table"]
    used, p = refs > 0, torch.arange(refs.numel(), device=GPU)
    n = used.sum()
    of, to = (used & (p >= n)).nonzero()[:, 0], (~used & (p < n)).nonzero()[:, 0]
    goes = p.index_copy(0, of, to)
    held = torch.arange(table.shape[1], device=GPU) < s["held"][:, None]
    table.copy_(torch.where(held & (table >= 0), goes[table.clamp(min=0).long()], table))
    refs[to] = refs[of]
    refs[of] = 0
    s["counts"][1] = n
    for x in s["caches"]:
        x[to] = x[of]


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    H, KV, hd, V = MODELS[case["model"]]
    op = case["op"]
    if op in ("fork", "compact"):
        return None  # nothing is computed: whole numbers, and values moved as they are
    if op == "rotary":
        out = {}
        for name in "qk":
            x = s[name].double()
            turn = torch.polar(torch.full((1, 1), s["magnitude"], device=GPU, dtype=torch.float64), s["positions"].double()[:, None] * s["frequencies"])
            r = x[..., :case["dims"]]
            z = r.unflatten(-1, (-1, 2)) if case["layout"] == "pairs" else r.unflatten(-1, (2, -1)).transpose(-1, -2)
            z = torch.view_as_real(torch.view_as_complex(z.contiguous()) * turn[:, None])
            r = z.flatten(-2) if case["layout"] == "pairs" else z.transpose(-1, -2).flatten(-2)
            out[name + "_out"] = torch.cat([r, x[..., case["dims"]:]], -1)
        return out
    if op == "beam":
        best = []
        for i in range(case["requests"]):
            mine = slice(i * case["beams"], (i + 1) * case["beams"])
            x = s["scores"][i].double()[:, None] + torch.log_softmax(s["logits"][mine].double(), -1)
            for b in s["finished"][i].nonzero()[:, 0]:
                x[b] = -math.inf
                x[b, 2] = s["scores"][i, b]
            best.append(x.flatten().topk(case["keep"]).values)
        return {"next": torch.stack(best), "parents": None, "tokens": None}
    page, block = case["page"], case["block"]
    if op == "append":
        codes, scales, row = s["codes"].double(), s["scales"].double(), 0
        x = torch.stack([s["new_k"], s["new_v"]]).double()
        for i, (new, length) in enumerate(_lengths(case)):
            a = length - new
            while a < length:  # block after block
                b = min(length, a // block * block + block)
                p, slot, nb = s["table"][i, a // page], a % page, a % page // block
                y = x[:, row:row + b - a].transpose(1, 2)  # [2, head, token, size]
                scale = (y.abs().amax((2, 3)) / 127).float().double()  # as it is stored
                if a % block:
                    scale = torch.maximum(scale, scales[:, p, nb])
                    old = codes[:, p, :, nb * block:slot]
                    codes[:, p, :, nb * block:slot] = (old * (scales[:, p, nb] / scale)[..., None, None]).round()
                scales[:, p, nb] = scale
                codes[:, p, :, slot:slot + b - a] = (y / scale[..., None, None]).round()
                row += b - a
                a = b
        scale = scales[:, s["written"]]
        return {"values": codes[:, s["written"]].unflatten(3, (page // block, block)) * scale.transpose(2, 3)[..., None, None], "scale": scale}
    row, out = 0, []
    for i, (new, length) in enumerate(_lengths(case)):
        mine = slice(row, row + new)
        row += new
        where = s["table"][i, :-(-length // page)].long()
        k, v = (c[where].double() * z[where].double().transpose(1, 2).repeat_interleave(block, 2)[..., None] for c, z in zip(s["codes"], s["scales"]))
        k, v = (y.permute(0, 2, 1, 3).reshape(-1, KV, hd)[:length] for y in (k, v))
        q = s["q"][mine].double() * s["scale"]
        o = torch.empty(new, H, hd, device=GPU, dtype=torch.float64)
        for h in range(H):
            kh, vh = k[:, h * KV // H].t().contiguous(), v[:, h * KV // H].contiguous()
            p = torch.arange(length - new, length, device=GPU)[:, None]
            seen = torch.arange(length, device=GPU)[None] <= p
            if case["window"]:
                seen &= torch.arange(length, device=GPU)[None] > p - case["window"]
            o[:, h] = torch.softmax((q[:, h].contiguous() @ kh).masked_fill(~seen, -math.inf), -1) @ vh
        out.append(o)
    return {"out": torch.cat(out)}
