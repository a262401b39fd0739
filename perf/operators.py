"""The operators of batched serving, as measurable cases.

A server that runs several sequences at once needs four things around a model's
matrices: new keys and values written into a cache of pages, attention of every
sequence's new tokens over its pages (single tokens and chunks of prompts in one
batch), attention over whole prompts packed one behind the other, and the log
probabilities of given tokens with the entropy and the most likely alternatives.
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


def listed():
    def append(name, model, seqs, new, length, page, src, ty):
        return {"name": name, "op": "append", "model": model, "seqs": seqs, "new": new, "chunks": seqs, "len": length, "page": page, "src": src, "type": ty}

    def paged(name, model, seqs, new, chunks, length, page, ty, window=0):
        return {"name": name, "op": "paged", "model": model, "seqs": seqs, "new": new, "chunks": chunks, "len": length, "page": page, "type": ty, "window": window}

    def packed(name, model, seqs, length, ty, window=0):
        return {"name": name, "op": "packed", "model": model, "seqs": seqs, "len": length, "type": ty, "window": window}

    def logprobs(name, model, rows, ty, top, targets):
        return {"name": name, "op": "logprobs", "model": model, "rows": rows, "type": ty, "top": top, "targets": targets}

    return [
        # one decode step of 61 sequences: a row each, behind very different lengths
        append("append-tokens-qwen3-30b-a3b", "qwen3-30b-a3b", 61, 1, 3000, 16, "f16", "f16"),
        # the prompts of a few new requests, from the f32 rows that the matrices give
        append("append-prompts-llama-3.1-8b", "llama-3.1-8b", 7, 1500, 1500, 64, "f32", "bf16"),
        # the smallest call: one short chat with a small model, 15 heads on 5
        paged("token-smollm2-360m-1x61", "smollm2-360m", 1, 1, 0, 61, 16, "f16"),
        # one decode step of a busy server, ragged lengths
        paged("token-llama-3.1-8b-48x4000", "llama-3.1-8b", 48, 1, 0, 4000, 16, "f16"),
        # the next token of one very long document
        paged("token-qwen3-30b-a3b-1x100003", "qwen3-30b-a3b", 1, 1, 0, 100003, 64, "bf16"),
        # a long prompt's chunks beside other sequences' single tokens in one batch
        paged("chunk-llama-3.1-8b-13x8200", "llama-3.1-8b", 13, 509, 3, 8200, 32, "bf16"),
        # a classifier's or scorer's batch of short prompts
        packed("packed-smollm2-360m-29x200", "smollm2-360m", 29, 200, "f16"),
        # long prompts packed: matrix work
        packed("packed-llama-3.1-8b-4x5000", "llama-3.1-8b", 4, 5000, "bf16"),
        # a window layer with 256-wide heads
        packed("packed-gemma-3-1b-5x2100-window", "gemma-3-1b", 5, 2100, "bf16", WINDOW),
        # the chosen token's log probability, 5 alternatives: one step of one chat
        logprobs("logprobs-qwen3-30b-a3b-1", "qwen3-30b-a3b", 1, "f32", 5, True),
        # perplexity over a text: every position's target
        logprobs("logprobs-llama-3.1-8b-512", "llama-3.1-8b", 512, "f32", 0, True),
        # distillation data: 20 alternatives of many positions from 16-bit logits
        logprobs("logprobs-qwen2.5-0.5b-1021", "qwen2.5-0.5b", 1021, "bf16", 20, True),
    ]


def draw(rng):
    def log(lo, hi):
        return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))

    most = max(_size(c) for c in listed())
    while True:
        op = rng.choice(["append", "paged", "paged", "paged", "packed", "packed", "logprobs", "logprobs"])
        model = rng.choice(sorted(MODELS))
        ty = rng.choice(["f16", "bf16"])
        window = WINDOW if model == "gemma-3-1b" and rng.random() < 0.5 else 0
        page = rng.choice([16, 32, 64, 128, 256])
        if op == "append":
            new = rng.choice([1, log(2, 1500)])
            seqs = log(1, 100)
            c = {"op": op, "model": model, "seqs": seqs, "new": new, "chunks": seqs, "len": max(new, log(1, 4000)), "page": page,
                 "src": rng.choice(["f32", ty]), "type": ty}
            good = seqs * new <= 20000
        elif op == "paged":
            new = rng.choice([1, 1, log(2, 8), log(9, 600)])
            seqs = log(1, 100)
            c = {"op": op, "model": model, "seqs": seqs, "new": new, "chunks": rng.randint(1, seqs) if new > 1 else 0,
                 "len": max(new, log(16, 100000)), "page": page, "type": ty, "window": window}
            good = seqs * c["len"] <= 200000 and seqs * new * c["len"] * MODELS[model][0] <= 2.5e9
        elif op == "packed":
            c = {"op": op, "model": model, "seqs": log(1, 64), "len": log(1, 6000), "type": ty, "window": window}
            good = c["seqs"] * c["len"] ** 2 * MODELS[model][0] <= 3.3e9
        else:
            c = {"op": op, "model": model, "rows": log(1, 1500), "type": rng.choice(["f32", "f32", "f16", "bf16"]),
                 "top": rng.choice([0, 1, 5, 20]), "targets": rng.random() < 0.8}
            good = c["targets"] or c["top"]
        if good and _size(c) <= most:
            return c


def _size(case):
    w = work(case)
    return max(w["bytes"], w["flops"] / 50)


def _lengths(case):
    """(new tokens, length with them) of every sequence; lengths from a tenth of the longest up, and the longest first"""
    r = random.Random(case["seqs"] * 1000003 + case["len"])
    n = case["seqs"]
    lens = [case["len"]] + [max(1, round(case["len"] * 10 ** -r.random())) for _ in range(n - 1)]
    if case["op"] == "packed":
        return [(x, x) for x in lens]
    if case["op"] == "append":  # every sequence brings about as much as the longest
        return [(min(x, max(1, round(case["new"] * r.uniform(0.5, 1.0)))) if case["new"] > 1 else 1, x) for x in lens]
    return [(min(case["new"], x) if i < case["chunks"] else 1, x) for i, x in enumerate(lens)]


def _pairs(new, length, window):
    """query and position pairs that one head computes"""
    seen = range(length - new + 1, length + 1)
    return sum(min(p, window) for p in seen) if window else new * (seen[0] + seen[-1]) // 2


def _read(new, length, window):
    """positions that at least one new token sees"""
    return min(length, window + new - 1) if window else length


def work(case):
    H, KV, hd, V = MODELS[case["model"]]
    if case["op"] == "logprobs":
        n = case["rows"] * V
        out = case["rows"] * (4 + 8 * case["top"] + (8 if case["targets"] else 0))
        return {"bytes": n * TYPES[case["type"]].itemsize + out, "flops": 4 * n}
    lens = _lengths(case)
    rows = sum(n for n, _ in lens)
    es = TYPES[case["type"]].itemsize
    if case["op"] == "append":
        return {"bytes": 2 * rows * KV * hd * (TYPES[case["src"]].itemsize + es) + 8 * rows, "flops": 0}
    positions = sum(_read(n, x, case["window"]) for n, x in lens)
    pairs = sum(_pairs(n, x, case["window"]) for n, x in lens)
    return {"bytes": (2 * rows * H * hd + 2 * positions * KV * hd) * es, "flops": 4 * hd * H * pairs}


def prepare(case, seed):
    g = torch.Generator(device=GPU).manual_seed(seed)
    H, KV, hd, V = MODELS[case["model"]]
    ty = TYPES[case["type"]]
    s = {"case": case}
    if case["op"] == "logprobs":
        # logits of a trained model: a wide body, and a few tokens that stand out
        n = case["rows"]
        x = torch.randn(n, V, device=GPU, generator=g) * 2.5 - 3
        at = torch.arange(40, device=GPU) * (V // 40) + torch.randint(0, V // 40, (n, 40), device=GPU, generator=g)
        x.scatter_(1, at, torch.rand(n, 40, device=GPU, generator=g) * 12 + 4)
        s["logits"] = x.to(ty)
        s["targets"] = torch.where(torch.rand(n, device=GPU, generator=g) < 0.8, at[:, 7], torch.randint(0, V, (n,), device=GPU, generator=g)).int() if case["targets"] else None
        s["logprob"] = torch.empty(n, device=GPU) if case["targets"] else None
        s["entropy"] = torch.empty(n, device=GPU)
        s["ids"] = torch.empty(n, case["top"], device=GPU, dtype=torch.int32) if case["top"] else None
        s["tops"] = torch.empty(n, case["top"], device=GPU) if case["top"] else None
    else:
        lens = _lengths(case)
        new = torch.tensor([n for n, _ in lens])
        s["starts"] = torch.cat([torch.zeros(1, dtype=torch.int64), new.cumsum(0)]).int().to(GPU)
        s["lens"] = torch.tensor([x for _, x in lens], dtype=torch.int32).to(GPU)
        s["max_new"], s["max_len"], s["rows"] = max(n for n, _ in lens), max(x for _, x in lens), int(new.sum())
    if case["op"] in ("append", "paged"):
        per = -(-s["max_len"] // case["page"])
        need = sum(-(-x // case["page"]) for _, x in lens)
        order = torch.randperm(need + 3, device=GPU, generator=g).int()
        used = torch.arange(per)[None] < -(-s["lens"].cpu()[:, None] // case["page"])
        table = torch.zeros(len(lens), per, dtype=torch.int32, device=GPU)
        table[used.to(GPU)] = order[:need]
        s["table"] = table
        # every KV head's rows of a page lie together, as in the backend's own cache
        s["k"], s["v"] = (torch.randn(need + 3, KV, case["page"], hd, device=GPU, generator=g).to(ty) for _ in range(2))
    if case["op"] == "append":
        # rows as the projections give them: keys and values of a token in one row
        src = torch.randn(s["rows"], 2 * KV, hd, device=GPU, generator=g).to(TYPES[case["src"]])
        s["new_k"], s["new_v"] = src[:, :KV], src[:, KV:]
    if case["op"] in ("paged", "packed"):
        if case["op"] == "packed":  # slices of the fused projection's rows
            qkv = torch.randn(s["rows"], H + 2 * KV, hd, device=GPU, generator=g)
            qkv[:, :H] *= 1.5
            qkv = qkv.to(ty)
            s["q"], s["new_k"], s["new_v"] = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        else:
            s["q"] = (torch.randn(s["rows"], H, hd, device=GPU, generator=g) * 1.5).to(ty)
        s["out"] = torch.empty(s["rows"], H, hd, device=GPU, dtype=ty)
        s["scale"] = 1 / math.sqrt(hd)
    if own:
        s["call"] = _call(s)
    return s


def _call(s):
    """The framework's call over the state's buffers, which a server makes at every layer and step."""
    from rust_interference_engine_amd import ops

    case = s["case"]
    if case["op"] == "logprobs":
        return ops.TokenLogprobs(s["logits"], targets=s["targets"], logprob=s["logprob"], entropy=s["entropy"], top_ids=s["ids"], top_logprobs=s["tops"])
    seqs = ops.Seqs(s["starts"], s["lens"], max_new=s["max_new"], max_len=s["max_len"])
    if case["op"] == "packed":
        return ops.PackedAttention(seqs, s["q"], s["new_k"], s["new_v"], s["out"], scale=s["scale"], window=case["window"])
    kv = ops.PagedKv(s["k"].transpose(1, 2), s["v"].transpose(1, 2), s["table"])
    if case["op"] == "append":
        return ops.PagedAppend(kv, seqs, s["new_k"], s["new_v"])
    return ops.PagedAttention(kv, seqs, s["q"], s["out"], scale=s["scale"], window=case["window"])


def run(s):
    if own:
        s["call"]()
    else:
        {"append": _append, "paged": _paged, "packed": _packed, "logprobs": _logprobs}[s["case"]["op"]](s)
    return {k: s[k] for k in {"append": ("k", "v"), "paged": ("out",), "packed": ("out",), "logprobs": ("logprob", "entropy", "ids", "tops")}[s["case"]["op"]]}


def _rows(s):
    """sequence and place within its new tokens of every row, and its position in the sequence"""
    starts, r = s["starts"].long(), torch.arange(s["rows"], device=GPU)
    seq = torch.searchsorted(starts, r, right=True) - 1
    at = r - starts[seq]
    return seq, at, (s["lens"].long() - starts[1:] + starts[:-1])[seq] + at


def _append(s):
    page = s["case"]["page"]
    seq, _, pos = _rows(s)
    p, slot = s["table"][seq, pos // page].long(), pos % page
    s["k"][p, :, slot] = s["new_k"].to(s["k"].dtype)
    s["v"][p, :, slot] = s["new_v"].to(s["v"].dtype)


def _attend(s, k, v):
    """k and v [sequence, KV head, position, size] in f32, padded to the longest; the new tokens padded likewise"""
    H, KV, hd, _ = MODELS[s["case"]["model"]]
    n, L, w = k.shape[0], k.shape[2], s["case"]["window"]
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


def _paged(s):
    def cached(pages):  # [sequence, page, head, slot, size] to [sequence, head, position, size]
        x = pages[s["table"].long()]
        return x.transpose(1, 2).flatten(2, 3).float()

    _attend(s, cached(s["k"]), cached(s["v"]))


def _packed(s):
    at = s["starts"].long()[:-1, None] + torch.arange(s["max_len"], device=GPU)
    at.clamp_(max=s["rows"] - 1)
    _attend(s, s["new_k"][at].transpose(1, 2).float(), s["new_v"][at].transpose(1, 2).float())


def _logprobs(s):
    x = s["logits"].float()
    V, top = x.shape[1], s["case"]["top"]
    d = x - x.amax(-1, keepdim=True)
    e = d.exp()
    total = e.sum(-1, keepdim=True)
    log_total = total.log()
    s["entropy"].copy_((log_total - (e * d).sum(-1, keepdim=True) / total)[:, 0])
    if s["targets"] is not None:
        s["logprob"].copy_((d.gather(1, s["targets"].long()[:, None]) - log_total)[:, 0])
    if top:
        # one whole-number key orders by value, then by index, the lowest first
        bits = (x + 0.0).view(torch.int32).long()
        key = (torch.where(bits >= 0, bits, bits ^ 0x7FFFFFFF) << 32) - torch.arange(V, device=GPU)
        ids = (-key.topk(top, -1).values) & 0xFFFFFFFF
        s["ids"].copy_(ids)
        s["tops"].copy_(d.gather(1, ids) - log_total)


def exact(case, seed):
    global own
    was, own = own, False
    s = prepare(case, seed)
    own = was
    if case["op"] == "logprobs":
        logprob, entropy, ids, tops = [], [], [], []
        for row in s["logits"].split(64):
            p = torch.log_softmax(row.double(), -1)
            entropy.append(-torch.xlogy(p.exp(), p.exp()).sum(-1))
            if case["targets"]:
                logprob.append(p[torch.arange(len(p)), s["targets"][64 * len(logprob):][:64].long()])
            if case["top"]:
                order = row.double().sort(dim=-1, descending=True, stable=True).indices[:, :case["top"]]
                ids.append(order.int())
                tops.append(torch.stack([a[b] for a, b in zip(p, order)]))
        return {"logprob": torch.cat(logprob) if logprob else None, "entropy": torch.cat(entropy),
                "ids": torch.cat(ids) if ids else None, "tops": torch.cat(tops) if tops else None}
    H, KV, hd, _ = MODELS[case["model"]]
    row, out = 0, []
    k, v = (s[c].clone() if case["op"] == "append" else None for c in "kv")
    for i, (new, length) in enumerate(_lengths(case)):
        mine = slice(row, row + new)
        row += new
        if case["op"] == "append":
            for t in range(new):
                page, slot = divmod(length - new + t, case["page"])
                at = s["table"][i, page]
                k[at, :, slot], v[at, :, slot] = s["new_k"][mine][t], s["new_v"][mine][t]
            continue
        if case["op"] == "packed":
            ks, vs = s["new_k"][mine].double(), s["new_v"][mine].double()
        else:
            where = s["table"][i, :-(-length // case["page"])].long()
            ks, vs = (s[c][where].permute(0, 2, 1, 3).reshape(-1, KV, hd)[:length].double() for c in "kv")
        q = s["q"][mine].double() * s["scale"]
        o = torch.empty(new, H, hd, device=GPU, dtype=torch.float64)
        for h in range(H):
            kh, vh = ks[:, h * KV // H].t().contiguous(), vs[:, h * KV // H].contiguous()
            for a in range(0, new, 2048):
                p = torch.arange(length - new + a, length - new + min(new, a + 2048), device=GPU)[:, None]
                seen = torch.arange(length, device=GPU)[None] <= p
                if case["window"]:
                    seen &= torch.arange(length, device=GPU)[None] > p - case["window"]
                score = (q[a:a + 2048, h].contiguous() @ kh).masked_fill(~seen, -math.inf)
                o[a:a + 2048, h] = torch.softmax(score, -1) @ vh
        out.append(o)
    return {"k": k, "v": v} if case["op"] == "append" else {"out": torch.cat(out)}
