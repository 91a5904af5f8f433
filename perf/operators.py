"""What is measured of the operators for batches of sequences over the paged cache.

The operators, each in its plain form (elementary torch operations in 32 bits) and as a program calls the library:

  norm-rope-store   qllm_k_qk_norm_rope_store: per-head norm of queries and keys, rotation by position, cache records
  attention         qllm_k_decode_attention: one new token per sequence over the cache, optional weight of each key
  evict             qllm_k_kv_evict: trims each sequence's cache to a budget by accumulated attention weight

The writer is measured with the exact F16 cache only: the codes of the Q8 and Q4H records are a rounding of computed
keys, whose borders two correct summation orders meet differently.  The readers are measured with every encoding.
"""
import math
import random

import numpy as np
import torch

own = False

F16, Q4H, Q8 = 0, 1, 2                      # cache encodings of the library
ROW = {"f32": (0, torch.float32, 4), "bf16": (1, torch.bfloat16, 2), "f16": (2, torch.float16, 2)}
PADDING = 0xFFFFFFFF                        # slot of a row that is not part of the batch
EPS, THETA = 1e-6, 1e6


def listed():
    return [
        # one stream's new token: the 27B geometry (40 query heads on 8), latency counts
        {"name": "norm-rope-store 1 row", "op": "norm", "rows": 1, "sequences": 1, "q": 40, "kv": 8, "hd": 128, "rot": 128,
         "row": "bf16", "page": 256, "first": 32768, "keys": False, "padding": 0},
        # a new token of 64 streams of the routed model (32 query heads on 4), a few places of the batch empty
        {"name": "norm-rope-store 64 streams", "op": "norm", "rows": 64, "sequences": 64, "q": 32, "kv": 4, "hd": 128, "rot": 128,
         "row": "f16", "page": 64, "first": 1000, "keys": False, "padding": 3},
        # prompts of uneven length, wide heads with a partial rotation, FP32 rows, keys handed on beside the records
        {"name": "norm-rope-store 517 f32 rows", "op": "norm", "rows": 517, "sequences": 5, "q": 12, "kv": 2, "hd": 256, "rot": 64,
         "row": "f32", "page": 16, "first": 0, "keys": True, "padding": 5},
        # a wide batch of prompt rows, 27B geometry
        {"name": "norm-rope-store 8192 rows", "op": "norm", "rows": 8192, "sequences": 16, "q": 40, "kv": 8, "hd": 128, "rot": 128,
         "row": "bf16", "page": 256, "first": 0, "keys": False, "padding": 0},
        # a short chat: the smallest reading of the cache
        {"name": "attention 1 x 1000", "op": "attention", "sequences": 1, "longest": 1000, "ragged": 0, "q": 40, "kv": 8, "hd": 128,
         "row": "bf16", "enc": F16, "page": 256, "weights": False},
        # the benchmark's stream: 32768 cached tokens in Q4H records
        {"name": "attention 1 x 32768 q4h", "op": "attention", "sequences": 1, "longest": 32768, "ragged": 0, "q": 40, "kv": 8, "hd": 128,
         "row": "bf16", "enc": Q4H, "page": 256, "weights": False},
        # 64 streams of very different lengths (empty ones among them), routed model, exact cache
        {"name": "attention 64 ragged", "op": "attention", "sequences": 64, "longest": 8192, "ragged": 11, "q": 32, "kv": 4, "hd": 128,
         "row": "bf16", "enc": F16, "page": 64, "weights": False},
        # the same for streams whose cache is trimmed by weight, Q8 records
        {"name": "attention 96 ragged weights", "op": "attention", "sequences": 96, "longest": 4500, "ragged": 12, "q": 40, "kv": 8, "hd": 128,
         "row": "f16", "enc": Q8, "page": 256, "weights": True},
        # no grouping, narrow heads, FP32 rows, long odd lengths, small pages
        {"name": "attention 7 x 20001 f32 weights", "op": "attention", "sequences": 7, "longest": 20001, "ragged": 13, "q": 16, "kv": 16, "hd": 64,
         "row": "f32", "enc": F16, "page": 16, "weights": True},
        # a full cache that takes one token a step
        {"name": "evict 1 of 4097", "op": "evict", "sequences": 1, "longest": 4097, "ragged": 0, "budget": 4096, "recent": 256, "sinks": 4,
         "kv": 8, "hd": 128, "enc": F16, "page": 256},
        # 48 streams trimmed after some hundred tokens each, Q4H records; some are still below the budget
        {"name": "evict 48 ragged q4h", "op": "evict", "sequences": 48, "longest": 6001, "ragged": 14, "budget": 4096, "recent": 512, "sinks": 4,
         "kv": 4, "hd": 128, "enc": Q4H, "page": 64},
        # long prompts cut to half
        {"name": "evict 8 x 32768 to half", "op": "evict", "sequences": 8, "longest": 32768, "ragged": 0, "budget": 16384, "recent": 1024, "sinks": 4,
         "kv": 8, "hd": 128, "enc": F16, "page": 256},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("norm", "attention", "evict")}
    while True:
        op = rng.choice(["norm", "attention", "attention", "evict"])
        hd = rng.choice([64, 128, 128, 192, 256])
        kv = rng.choice([1, 2, 3, 4, 5, 8, 16])
        page = rng.choice([16, 48, 64, 256])
        if op == "norm":
            sequences = _spread(rng, 1, 64)
            rows = max(sequences, _spread(rng, 1, 8192))
            c = {"op": op, "rows": rows, "sequences": sequences, "q": kv * rng.choice([1, 2, 5, 6, 8]), "kv": kv, "hd": hd,
                 "rot": rng.choice([hd, hd // 2, hd // 4, 0]), "row": rng.choice(["bf16", "bf16", "f16", "f32"]), "page": page,
                 "first": _spread(rng, 1, 200000) - 1, "keys": rng.random() < 0.3, "padding": rng.choice([0, 0, min(3, rows - 1)])}
        elif op == "attention":
            sequences = _spread(rng, 1, 128)
            c = {"op": op, "sequences": sequences, "longest": _spread(rng, 1, 131072), "ragged": rng.choice([0, rng.randrange(1, 1000)]),
                 "q": kv * rng.choice([1, 2, 5, 6, 8, 8, 12]), "kv": kv, "hd": hd, "row": rng.choice(["bf16", "bf16", "f16", "f32"]),
                 "enc": rng.choice([F16, Q4H, Q8]), "page": page, "weights": rng.random() < 0.4}
        else:
            longest = _spread(rng, 2, 131072)
            budget = max(1, int(longest * rng.choice([0.25, 0.5, 0.8, 0.97])))
            recent = rng.choice([0, 1, budget // 8, budget // 2])
            c = {"op": op, "sequences": _spread(rng, 1, 64), "longest": longest, "ragged": rng.choice([0, rng.randrange(1, 1000)]),
                 "budget": budget, "recent": recent, "sinks": min(4, budget - recent), "kv": kv, "hd": hd,
                 "enc": rng.choice([F16, Q4H, Q8]), "page": page}
        if _cost(c) <= most[op]:
            return c


def _cost(c):
    """What limits a drawn case: the work, and what the plain form holds (padded to the longest)."""
    if c["op"] == "norm":
        return work(c)["bytes"]
    return c["sequences"] * c["longest"] * c["kv"] * c["hd"]


# ------------------------------------------------------------------------------- the cache

def _record_bytes(enc, hd):
    return {F16: 2 * hd, Q4H: hd // 2 + 2, Q8: hd + 2}[enc]


def _lengths(c):
    """Cached tokens of each sequence: all `longest`, or spread, with a sequence of none and one of a single token."""
    n, top = c["sequences"], c["longest"]
    if not c["ragged"]:
        return [top] * n
    r = random.Random(c["ragged"])
    got = [max(1, int(top * r.random() ** 0.7)) for _ in range(n)]
    got[0] = top
    if n > 2:
        got[1], got[2] = 0, 1
    r.shuffle(got)
    return got


class Cache:
    """A pool of pages (one layer each) and the page tables of a batch: page i of a sequence lies anywhere in the pool."""

    def __init__(self, g, sequences, tokens, page, enc, kv, hd, fill):
        self.sequences, self.page, self.enc, self.kv, self.hd = sequences, page, enc, kv, hd
        self.pages = -(-tokens // page)
        self.page_bytes = 2 * page * kv * _record_bytes(enc, hd)
        total = sequences * self.pages
        self.pool = torch.zeros(total, self.page_bytes, dtype=torch.uint8, device="cuda")
        self.index = torch.randperm(total, generator=g, device="cuda").view(sequences, self.pages)
        self.tables = (self.pool.data_ptr() + self.index * self.page_bytes).contiguous()
        if fill:
            self._fill(g)

    def _fill(self, g):
        if self.enc == F16:
            self.pool.view(torch.float16).normal_(generator=g)
            return
        for codes, scales in self.sections():
            if self.enc == Q8:
                codes.random_(1, 256, generator=g)               # two's complement -127..127
                codes[codes == 128] = 0
                scales.uniform_(0.01, 0.03, generator=g)
            else:
                nibbles = torch.randint(-7, 8, (2, *codes.shape), generator=g, device="cuda", dtype=torch.int8) & 15
                codes.copy_((nibbles[0] | (nibbles[1] << 4)).view(torch.uint8))
                scales.uniform_(0.15, 0.35, generator=g)

    def sections(self):
        """(K, V) as views of the pool.  F16: values [P, pt, kv, hd]; else (codes, scales): Q8 [P, pt, kv, hd] and
        [P, pt, kv]; Q4H [P, kv, pt, hd / 2] and [P, kv, pt]."""
        p, pt, kv, hd = self.pool, self.page, self.kv, self.hd
        if self.enc == F16:
            both = p.view(torch.float16).view(-1, 2, pt, kv, hd)
            return both[:, 0], both[:, 1]
        if self.enc == Q8:
            both = p.view(-1, 2, pt, kv, hd + 2)
            halves = p.view(torch.float16).view(-1, 2, pt, kv, hd // 2 + 1)
            return tuple((both[:, i, :, :, :hd], halves[:, i, :, :, hd // 2]) for i in (0, 1))
        records = pt * kv
        at = [0, records * hd // 2, records * (hd // 2 + 2), records * (hd + 2)]
        return tuple((p[:, at[2 * i]:at[2 * i + 1]].view(-1, kv, pt, hd // 2),
                      p.view(torch.float16)[:, at[2 * i + 1] // 2:at[2 * i + 1] // 2 + records].view(-1, kv, pt)) for i in (0, 1))

    def values(self, dtype):
        """Dequantised (K, V) of every sequence: [sequences, kv, pages * page, hd]."""
        got = []
        for part in self.sections():
            if self.enc == F16:
                x = part[self.index].to(dtype).permute(0, 3, 1, 2, 4)
            else:
                codes, scales = part[0][self.index], part[1][self.index].to(dtype)
                if self.enc == Q8:
                    x = (codes.view(torch.int8).to(dtype) * scales[..., None]).permute(0, 3, 1, 2, 4)
                else:
                    low, high = (codes << 4).view(torch.int8) >> 4, codes.view(torch.int8) >> 4
                    x = (torch.stack((low, high), -1).flatten(-2).to(dtype) * scales[..., None]).permute(0, 2, 1, 3, 4)
            got.append(x.flatten(2, 3))
        return got

    def descriptor(self, ql):
        return ql.KvBatch(self.tables.data_ptr(), 0, self.sequences, self.pages, self.page, self.enc, self.kv, self.hd)


# ------------------------------------------------------------------------------- inputs

def _int32(values):
    return torch.tensor([v - (1 << 32) if v >= 1 << 31 else v for v in values], dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = {"case": c}
    if c["op"] == "norm":
        rows, width = c["rows"], (c["q"] + 2 * c["kv"]) * c["hd"]
        dtype = ROW[c["row"]][1]
        real = rows - c["padding"]
        # rows of the sequences one after the other, each continuing its cache at a slot of its own
        each = [real // c["sequences"] + (i < real % c["sequences"]) for i in range(c["sequences"])]
        r = random.Random(seed)
        start = [r.randrange(c["page"]) for _ in each]
        sequence, slot, position = [], [], []
        for i, n in enumerate(each):
            sequence += [i] * n
            slot += range(start[i], start[i] + n)
            position += range(c["first"] + start[i], c["first"] + start[i] + n)
        sequence += [0] * c["padding"]
        slot += [PADDING] * c["padding"]
        position += [0] * c["padding"]
        s["cache"] = Cache(g, c["sequences"], max(a + n for a, n in zip(start, each)), c["page"], F16, c["kv"], c["hd"], False)
        s["qkv"] = torch.randn(rows, width, generator=g, device="cuda").to(dtype)
        s["q_norm"] = 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")
        s["k_norm"] = 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda")
        half = c["rot"] // 2
        s["inv_freq"] = torch.tensor([THETA ** (-i / half) for i in range(half)] or [0.0], dtype=torch.float32, device="cuda")
        s["sequence"], s["slot"], s["position"] = _int32(sequence), _int32(slot), _int32(position)
        s["query"] = torch.zeros(rows, c["q"] * c["hd"], dtype=dtype, device="cuda")
        s["key"] = torch.zeros(rows, c["kv"] * c["hd"], dtype=dtype, device="cuda") if c["keys"] else None
        s["slot_positions"] = torch.zeros(c["sequences"], c["kv"], s["cache"].pages * c["page"], dtype=torch.int32, device="cuda")
        return s
    lengths = _lengths(c)
    top = max(lengths)
    s["cache"] = Cache(g, c["sequences"], top, c["page"], c["enc"], c["kv"], c["hd"], True)
    s["lengths"] = _int32(lengths)
    slots = s["cache"].pages * c["page"]
    if c["op"] == "attention":
        dtype = ROW[c["row"]][1]
        s["query"] = (2 * torch.randn(c["sequences"], c["q"] * c["hd"], generator=g, device="cuda")).to(dtype)
        s["out"] = torch.zeros_like(s["query"])
        if c["weights"]:
            s["weights"] = torch.rand(c["sequences"], c["kv"], slots, generator=g, device="cuda")
            s["weights_out"] = torch.zeros_like(s["weights"])
        return s
    # accumulated weights are heavy-tailed; the slots below the budget are no longer in the order of their positions
    shape = (c["sequences"], c["kv"], slots)
    s["weights"] = torch.exp(2 * torch.randn(shape, generator=g, device="cuda"))
    s["weights_out"] = torch.zeros_like(s["weights"])
    base = torch.arange(slots, device="cuda", dtype=torch.int32).expand(shape).clone()
    held = min(c["budget"], slots)
    base[..., :held] = base[..., torch.randperm(held, generator=g, device="cuda")]
    s["positions"] = base
    s["positions_out"] = torch.zeros_like(base)
    s["next"] = s["lengths"].clone()
    s["lengths_out"] = torch.zeros_like(s["lengths"])
    return s


# ------------------------------------------------------------------------------- one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return {"norm": _own_norm, "attention": _own_attention, "evict": _own_evict}[op](state)
    return {"norm": _plain_norm, "attention": _plain_attention, "evict": _plain_evict}[op](state)


def _library(state):
    from quantum_llm_b200 import lib as ql
    if "descriptor" not in state:
        state["descriptor"] = state["cache"].descriptor(ql)
    return ql, ql.load(), state["descriptor"]


def _workspace(state, size):
    """The caller's scratch memory, made at the first call and kept, as a program does."""
    if "workspace" not in state:
        state["workspace"] = torch.empty(max(16, size()), dtype=torch.uint8, device="cuda")
    return state["workspace"]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _ptr(x):
    return None if x is None else x.data_ptr()


def _outputs_norm(s):
    return {"query": s["query"], "key": s["key"], "cache": s["cache"].pool.view(torch.float16), "positions": s["slot_positions"]}


def _own_norm(s):
    ql, L, cache = _library(s)
    c = s["case"]
    ql.check(L.qllm_k_qk_norm_rope_store(
        cache, ROW[c["row"]][0], _ptr(s["qkv"]), s["qkv"].stride(0), c["rows"], c["q"], c["rot"], _ptr(s["q_norm"]), _ptr(s["k_norm"]), EPS,
        _ptr(s["inv_freq"]), _ptr(s["position"]), _ptr(s["sequence"]), _ptr(s["slot"]), _ptr(s["query"]), s["query"].stride(0),
        _ptr(s["key"]), c["kv"] * c["hd"] if c["keys"] else 0, _ptr(s["slot_positions"]), s["slot_positions"].stride(1), _stream()))
    return _outputs_norm(s)


def _own_attention(s):
    ql, L, cache = _library(s)
    c = s["case"]
    weights = c["weights"]
    ws = _workspace(s, lambda: L.qllm_k_decode_attention_workspace_bytes(cache, c["q"], int(weights)))
    ql.check(L.qllm_k_decode_attention(
        cache, ROW[c["row"]][0], _ptr(s["query"]), s["query"].stride(0), _ptr(s["lengths"]), c["q"], c["hd"] ** -0.5,
        _ptr(s["weights"]) if weights else None, _ptr(s["weights_out"]) if weights else None,
        s["weights"].stride(1) if weights else 0, _ptr(s["out"]), s["out"].stride(0), _ptr(ws), ws.numel(), _stream()))
    return {"out": s["out"], "weights": s["weights_out"] if weights else None}


def _own_evict(s):
    ql, L, cache = _library(s)
    c = s["case"]
    ws = _workspace(s, lambda: L.qllm_k_kv_evict_workspace_bytes(cache, c["budget"]))
    ql.check(L.qllm_k_kv_evict(
        cache, _ptr(s["lengths"]), _ptr(s["lengths_out"]), _ptr(s["next"]), c["budget"], c["recent"], c["sinks"], _ptr(s["weights"]),
        _ptr(s["weights_out"]), _ptr(s["positions"]), _ptr(s["positions_out"]), s["weights"].stride(1), _ptr(ws), ws.numel(), _stream()))
    return _outputs_evict(s)


def _outputs_evict(s):
    return {"cache": s["cache"].pool.view(torch.int64), "weights": s["weights_out"], "positions": s["positions_out"], "lengths": s["lengths_out"]}


def _plain_norm(s):
    c = s["case"]
    rows, q, kv, hd, rot = c["rows"], c["q"], c["kv"], c["hd"], c["rot"]
    x = s["qkv"].float().view(rows, q + 2 * kv, hd)
    qk, v = x[:, :q + kv], x[:, q + kv:]
    w = torch.cat((s["q_norm"].expand(q, hd), s["k_norm"].expand(kv, hd)))
    qk = qk / torch.sqrt((qk * qk).mean(-1, keepdim=True) + EPS) * w
    if rot:
        angle = s["position"].double()[:, None] * s["inv_freq"].double()
        cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
        a, b = qk[..., :rot // 2], qk[..., rot // 2:rot]
        qk = torch.cat((a * cos - b * sin, b * cos + a * sin, qk[..., rot:]), -1)
    live = rows - c["padding"]           # the padding stands at the end
    s["query"][:live] = qk[:live, :q].reshape(live, q * hd).to(s["query"].dtype)
    if c["keys"]:
        s["key"][:live] = qk[:live, q:].reshape(live, kv * hd).to(s["key"].dtype)
    cache = s["cache"]
    slot, sequence = s["slot"][:live].long(), s["sequence"][:live].long()
    page, place = cache.index[sequence, slot // cache.page], slot % cache.page
    keys, values = cache.sections()
    keys[page, place] = qk[:live, q:].half()
    values[page, place] = v[:live].half()
    s["slot_positions"][sequence, :, slot] = s["position"][:live, None].expand(live, kv)
    return _outputs_norm(s)


def _plain_attention(s):
    c = s["case"]
    n, q, kv, hd = c["sequences"], c["q"], c["kv"], c["hd"]
    keys, values = s["cache"].values(torch.float32)
    slots = keys.shape[2]
    query = s["query"].float().view(n, kv, q // kv, hd)
    z = query @ keys.transpose(2, 3) * hd ** -0.5
    live = (torch.arange(slots, device="cuda") < s["lengths"][:, None])[:, None, None]
    z = z.masked_fill(~live, -math.inf)
    p = (z - z.amax(-1, keepdim=True).clamp_min(-3e38)).exp()
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = (p @ values).reshape(n, q * hd).to(s["query"].dtype)
    if not c["weights"]:
        return {"out": out, "weights": None}
    weights = torch.where(live[:, :, 0], s["weights"] + p.sum(2), torch.zeros_like(s["weights"]))
    return {"out": out, "weights": weights}


def _plain_evict(s):
    c = s["case"]
    cache, kv = s["cache"], c["kv"]
    w, pos = s["weights"], s["positions"].long()
    slots = torch.arange(w.shape[2], device="cuda").expand(w.shape)
    n = s["lengths"].long()[:, None, None]
    m = n.clamp_max(c["budget"])
    safe = (pos + c["recent"] >= s["next"].long()[:, None, None]) | (pos < c["sinks"])
    rank = torch.where(slots < n, 1 + safe.long(), torch.zeros_like(pos))
    order = torch.where(w.isnan(), torch.full_like(w, -math.inf), w).sort(dim=-1, descending=True, stable=True).indices
    order = order.gather(-1, rank.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices)
    kept = torch.zeros_like(safe).scatter(-1, order, slots < m)
    # the i-th freed slot below m takes the i-th kept one at or above m
    hole, mover = (slots < m) & ~kept, (slots >= m) & kept
    movers = torch.where(mover, slots, slots + w.shape[2]).sort(-1).values
    source = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slots)
    source = torch.where(slots < m, source, slots)
    s["weights_out"].copy_(torch.where(slots < m, w.gather(-1, source), torch.zeros_like(w)))
    s["positions_out"].copy_(torch.where(slots < m, s["positions"].gather(-1, source), torch.zeros_like(s["positions"])))
    s["lengths_out"].copy_(m[:, 0, 0])
    held = min(c["budget"], w.shape[2])
    src, dst = source[..., :held], slots[..., :held]
    row = torch.arange(c["sequences"], device="cuda")[:, None, None]
    head = torch.arange(kv, device="cuda")[None, :, None]
    spot = lambda t: (cache.index[row, t // cache.page], t % cache.page)  # noqa: E731
    (page_s, place_s), (page_d, place_d) = spot(src), spot(dst)
    for part in cache.sections():
        if cache.enc == F16:
            part[page_d, place_d, head] = part[page_s, place_s, head]
        elif cache.enc == Q8:
            for x in part:
                x[page_d, place_d, head] = x[page_s, place_s, head]
        else:
            for x in part:
                x[page_d, head, place_d] = x[page_s, head, place_s]
    return _outputs_evict(s)


# ------------------------------------------------------------------------------- what a pass cannot do without

def work(case):
    c = case
    hd, kv = c["hd"], c["kv"]
    if c["op"] == "norm":
        rows, size = c["rows"] - c["padding"], ROW[c["row"]][2]
        values = rows * (2 * c["q"] + 2 * kv + (kv if c["keys"] else 0)) * hd * size
        return {"bytes": values + rows * kv * (4 * hd + 4) + rows * 12, "flops": rows * (c["q"] + kv) * hd * 8}
    lengths = _lengths(c)
    record = _record_bytes(c["enc"], hd)
    if c["op"] == "attention":
        tokens, size = sum(lengths), ROW[c["row"]][2]
        return {"bytes": tokens * kv * (2 * record + (8 if c["weights"] else 0)) + 2 * c["sequences"] * c["q"] * hd * size,
                "flops": 4 * tokens * c["q"] * hd}
    total, moved = 0.0, 0.0
    for n in lengths:
        m = min(n, c["budget"])
        total += 8 * n + 8 * m + 4 * (n - m)
        if n > m:
            # of the slots at or above m the recent ones are kept, of the others the share that the budget leaves
            late = min(c["recent"], n - m)
            safe = c["recent"] + c["sinks"]
            moved += late + (n - m - late) * max(0, m - safe) / max(1, n - safe)
    return {"bytes": kv * (total + moved * 4 * record) + 12 * c["sequences"], "flops": kv * sum(lengths)}


# ------------------------------------------------------------------------------- the definition in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _exact_norm, "attention": _exact_attention, "evict": _exact_evict}[case["op"]](s)


def _exact_norm(s):
    c = s["case"]
    q, kv, hd, half = c["q"], c["kv"], c["hd"], c["rot"] // 2
    live = c["rows"] - c["padding"]
    x = s["qkv"].double().reshape(c["rows"], -1, hd)[:live]
    heads = []
    for w, part in ((s["q_norm"], x[:, :q]), (s["k_norm"], x[:, q:q + kv])):
        y = part * w.double() * (part.square().sum(-1, keepdim=True) / hd + EPS).rsqrt()
        if half:
            turn = torch.polar(torch.ones(live, half, dtype=torch.float64, device="cuda"),
                               torch.outer(s["position"][:live].double(), s["inv_freq"].double()))
            z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn[:, None]
            y = torch.cat((z.real, z.imag, y[..., 2 * half:]), -1)
        heads.append(y)
    cache = s["cache"]
    query = torch.zeros(c["rows"], q * hd, dtype=torch.float64, device="cuda")
    query[:live] = heads[0].flatten(1)
    key = None
    if c["keys"]:
        key = torch.zeros(c["rows"], kv * hd, dtype=torch.float64, device="cuda")
        key[:live] = heads[1].flatten(1)
    pool = torch.zeros(cache.pool.shape[0] * 2, c["page"], kv * hd, dtype=torch.float64, device="cuda")
    slot, sequence = s["slot"][:live].long(), s["sequence"][:live].long()
    page = cache.index[sequence, slot // c["page"]]
    pool[2 * page, slot % c["page"]] = heads[1].flatten(1)
    pool[2 * page + 1, slot % c["page"]] = x[:, q + kv:].flatten(1)
    return {"query": query, "key": key, "cache": pool.view(cache.pool.shape[0], -1), "positions": None}


def _exact_attention(s):
    c = s["case"]
    cache, group = s["cache"], c["q"] // c["kv"]
    out = torch.zeros(c["sequences"], c["kv"], group, c["hd"], dtype=torch.float64, device="cuda")
    weights = torch.zeros_like(s["weights"], dtype=torch.float64) if c["weights"] else None
    index, n = cache.index, 0
    for i, n in enumerate(_lengths(c)):
        if not n:
            continue
        cache.index = index[i:i + 1]
        keys, values = (t[0, :, :n] for t in cache.values(torch.float64))
        z = torch.einsum("hgd,htd->hgt", s["query"][i].double().view(c["kv"], group, c["hd"]), keys) / math.sqrt(c["hd"])
        p = torch.softmax(z, -1)
        out[i] = torch.einsum("hgt,htd->hgd", p, values)
        if weights is not None:
            weights[i, :, :n] = s["weights"][i, :, :n].double() + p.sum(1)
    cache.index = index
    return {"out": out.view(c["sequences"], -1), "weights": weights}


def _exact_evict(s):
    c = s["case"]
    w, pos = s["weights"].cpu().numpy(), s["positions"].cpu().numpy().astype(np.int64)
    weights, positions = np.zeros(w.shape), np.zeros(w.shape, np.int64)
    lengths = _lengths(c)
    for i, n in enumerate(lengths):
        m = min(n, c["budget"])
        for h in range(c["kv"]):
            a, p = w[i, h, :n], pos[i, h, :n]
            plain = ~((p >= n - c["recent"]) | (p < c["sinks"]))
            best = np.lexsort((np.arange(n), -a, plain))[:m]
            stay, move = best[best < m], np.sort(best[best >= m])
            source = np.arange(m)
            source[np.setdiff1d(np.arange(m), stay)] = move
            weights[i, h, :m], positions[i, h, :m] = a[source], p[source]
    return {"cache": None, "weights": torch.from_numpy(weights), "positions": None, "lengths": None}
