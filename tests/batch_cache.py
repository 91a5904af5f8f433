"""A paged cache for the tests of the batched cache operators: pages of several layers scattered over a
pool, with the records read and written by plain torch code from the layouts in include/qllm_b200.h."""
import torch

from quantum_llm_b200 import lib as ql

F16, Q4H, Q8 = ql.KV_F16, ql.KV_Q4H, ql.KV_Q8
TYPES = {torch.float32: ql.ROW_F32, torch.bfloat16: ql.ROW_BF16, torch.float16: ql.ROW_F16}
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def layer_bytes(enc, page, kv, hd):
    return 2 * page * kv * {F16: 2 * hd, Q4H: hd // 2 + 2, Q8: hd + 2}[enc]


def raw(x):
    """The bytes of x, the last dimension's one after the other."""
    return torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x).view(torch.uint8)


class PagedCache:
    """`layers` layers to a page; the operators work on layer `layer`.  absent: [(sequence, page)] without a page."""

    def __init__(self, sequences, pages, page, enc, kv, hd, layers=1, layer=0, seed=0, absent=(), fill=True):
        self.sequences, self.pages, self.page, self.enc, self.kv, self.hd = sequences, pages, page, enc, kv, hd
        self.bytes = layer_bytes(enc, page, kv, hd)
        self.layer = layer
        g = torch.Generator(device="cuda").manual_seed(seed)
        total = sequences * pages
        self.pool = torch.randint(0, 256, (total, layers * self.bytes), generator=g, device="cuda", dtype=torch.uint8)
        self.index = torch.randperm(total, generator=g, device="cuda").view(sequences, pages)
        self.tables = (self.pool.data_ptr() + self.index * (layers * self.bytes)).contiguous()
        for s, p in absent:
            self.tables[s, p] = 0
        if fill:
            self.fill(g)

    @property
    def capacity(self):
        return self.pages * self.page

    def mine(self):
        """This layer's bytes of every page, [pages of the pool, bytes], as a view."""
        return self.pool[:, self.layer * self.bytes:(self.layer + 1) * self.bytes]

    def parts(self, pages):
        """(codes or values, scales or None) of K and V over contiguous layer bytes [P, bytes], every tensor
        indexed [P, place, kv head]."""
        n, pt, kv, hd = pages.shape[0], self.page, self.kv, self.hd
        half = self.bytes // 2
        got = []
        for b in (pages[:, :half].contiguous(), pages[:, half:].contiguous()):
            if self.enc == F16:
                got.append((b.view(torch.float16).view(n, pt, kv, hd), None))
            elif self.enc == Q8:
                b = b.view(n, pt, kv, hd + 2)
                got.append((b[..., :hd].contiguous().view(torch.int8), b[..., hd:].contiguous().view(torch.float16)[..., 0]))
            else:
                codes, scales = b[:, :pt * kv * hd // 2].contiguous(), b[:, pt * kv * hd // 2:].contiguous()
                got.append((codes.view(n, kv, pt, hd // 2).transpose(1, 2), scales.view(torch.float16).view(n, kv, pt).transpose(1, 2)))
        return got

    def fill(self, g, spread=1.0):
        """Random records that a writer could have made."""
        m = self.mine()
        if self.enc == F16:
            m.copy_((torch.randn(m.shape[0], self.bytes // 2, generator=g, device="cuda") * spread).half().view(torch.uint8))
            return
        records = self.page * self.kv
        for half in (0, self.bytes // 2):
            n = m.shape[0]
            if self.enc == Q8:
                codes = torch.randint(-127, 128, (n, records, self.hd), generator=g, device="cuda", dtype=torch.int8).view(torch.uint8)
                scale = (0.01 + 0.02 * torch.rand(n, records, 1, generator=g, device="cuda")).half().view(torch.uint8)
                b = torch.cat((codes, scale), -1).view(n, -1)
            else:
                low, high = (torch.randint(-7, 8, (n, records * self.hd // 2), generator=g, device="cuda", dtype=torch.int8) & 15 for _ in range(2))
                scale = (0.15 + 0.2 * torch.rand(n, records, generator=g, device="cuda")).half().view(torch.uint8)
                b = torch.cat(((low | (high << 4)).view(torch.uint8), scale), -1)
            m[:, half:half + self.bytes // 2] = b

    def values(self, s, n=None):
        """(K, V) of sequence s in FP64, [slots, kv heads, head_dim], and which slots have a page."""
        n = self.capacity if n is None else n
        there = (self.tables[s] != 0).repeat_interleave(self.page)[:n]
        got = []
        for codes, scales in self.parts(self.mine()[self.index[s]]):
            x = codes
            if self.enc == Q4H:
                signed = lambda v: torch.where(v >= 8, v - 16, v)  # noqa: E731
                x = torch.stack((signed((codes & 15).to(torch.int8)), signed((codes >> 4).to(torch.int8))), -1).flatten(-2)
            x = x.double()
            if scales is not None:
                x = x * scales.double()[..., None]
            got.append(x.reshape(self.capacity, self.kv, self.hd)[:n])
        return got[0], got[1], there

    def records(self):
        """Raw bytes of every record, [sequences, slots, kv heads, bytes of K and V], for equality."""
        per = []
        for codes, scales in self.parts(self.mine()):
            per.append(raw(codes))
            if scales is not None:
                per.append(raw(scales[..., None]))
        x = torch.cat(per, -1)[self.index]
        return x.reshape(self.sequences, self.capacity, self.kv, -1)

    def descriptor(self):
        return ql.KvBatch(self.tables.data_ptr(), self.layer * self.bytes, self.sequences, self.pages, self.page, self.enc, self.kv, self.hd)


def u32(values):
    return torch.tensor([v - (1 << 32) if v >= 1 << 31 else v for v in values], dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


def ptr(x):
    return None if x is None else x.data_ptr()


def norm_rope_store(cache, qkv, q_heads, rot, q_norm, k_norm, inv, positions, sequence, slot, query, key=None, slot_positions=None,
                    eps=1e-6):
    L = ql.load()
    ql.check(L.qllm_k_qk_norm_rope_store(
        cache.descriptor(), TYPES[qkv.dtype], ptr(qkv), qkv.stride(0), qkv.shape[0], q_heads, rot, ptr(q_norm), ptr(k_norm), eps, ptr(inv),
        ptr(positions), ptr(sequence), ptr(slot), ptr(query), query.stride(0), ptr(key), key.stride(0) if key is not None else 0,
        ptr(slot_positions), slot_positions.stride(1) if slot_positions is not None else 0, stream()))


def attention_workspace(cache, q_heads, weights):
    size = ql.load().qllm_k_decode_attention_workspace_bytes(cache.descriptor(), q_heads, int(weights))
    return torch.full((max(size, 16),), 0xA5, dtype=torch.uint8, device="cuda")   # its content must not matter


def decode_attention(cache, query, lengths, q_heads, scale, out, weights_in=None, weights_out=None, workspace=None):
    ws = attention_workspace(cache, q_heads, weights_out is not None) if workspace is None else workspace
    ql.check(ql.load().qllm_k_decode_attention(
        cache.descriptor(), TYPES[query.dtype], ptr(query), query.stride(0), ptr(lengths), q_heads, scale, ptr(weights_in),
        ptr(weights_out), weights_out.stride(1) if weights_out is not None else 0, ptr(out), out.stride(0), ptr(ws), ws.numel(), stream()))
    return ws   # the caller keeps it while the call may run


def evict_workspace(cache, budget):
    size = ql.load().qllm_k_kv_evict_workspace_bytes(cache.descriptor(), budget)
    return torch.full((max(size, 16),), 0xA5, dtype=torch.uint8, device="cuda")


def evict(cache, lengths_in, lengths_out, following, budget, recent, sinks, w_in, w_out, p_in, p_out, workspace=None):
    ws = evict_workspace(cache, budget) if workspace is None else workspace
    ql.check(ql.load().qllm_k_kv_evict(
        cache.descriptor(), ptr(lengths_in), ptr(lengths_out), ptr(following), budget, recent, sinks, ptr(w_in), ptr(w_out), ptr(p_in),
        ptr(p_out), w_in.stride(1), ptr(ws), ws.numel(), stream()))
    return ws


# ---------------------------------------------------------------- the definitions in 64 bits

def exact_norm_rope(x, q_heads, kv, hd, rot, q_norm, k_norm, inv, positions, eps=1e-6):
    """(query heads, key heads, bound on the magnitudes that a rotation adds up), all FP64 [rows, heads, hd]."""
    x = x.double().view(x.shape[0], -1, hd)
    w = torch.cat((q_norm.double().expand(q_heads, hd), k_norm.double().expand(kv, hd)))
    n = x[:, :q_heads + kv]
    n = n / (n.pow(2).mean(-1, keepdim=True) + eps).sqrt() * w
    y, size = n.clone(), n.abs()
    half = rot // 2
    if half:
        a = torch.tensor([float(p) for p in positions], dtype=torch.float64, device="cuda")[:, None] * inv.double()[:half]
        cos, sin = a.cos()[:, None], a.sin()[:, None]
        low, high = n[..., :half], n[..., half:rot]
        y[..., :half] = low * cos - high * sin
        y[..., half:rot] = high * cos + low * sin
        size[..., :half] = size[..., half:rot] = low.abs() + high.abs()
    return y[:, :q_heads], y[:, q_heads:], size


def exact_attention(cache, s, n, q, q_heads, scale):
    """Of one sequence: (out [q_heads, hd], p [q_heads, n], sum p|V|, largest sum |q||K| scale, sum |V|)."""
    hd, group = cache.hd, q_heads // cache.kv
    k, v, there = cache.values(s, n)
    q = q.double().view(cache.kv, group, hd)
    z = torch.einsum("hgd,thd->hgt", q, k) * scale
    z = z.masked_fill(~there, float("-inf"))
    size = (torch.einsum("hgd,thd->hgt", q.abs(), k.abs()) * abs(scale)).masked_fill(~there, 0.0)
    size = size.amax(-1) if n else size.sum(-1)
    if not bool(there.any()):
        p = torch.zeros_like(z)
    else:
        p = torch.softmax(z, -1)
    v = torch.where(there[:, None, None], v, torch.zeros_like(v))   # what an absent or masked slot holds does not count
    out = torch.einsum("hgt,thd->hgd", p, v)
    spread = torch.einsum("hgt,thd->hgd", p, v.abs())
    return out.reshape(q_heads, hd), p.reshape(q_heads, n), spread.reshape(q_heads, hd), size.reshape(q_heads), \
        v.abs().sum(0).repeat_interleave(group, 0)


def exact_evict(w, p, n, following, budget, recent, sinks):
    """Of one (sequence, kv head), in Python: (source slot of each kept slot, freed slots, kept slots at or above m)."""
    m = min(n, budget)

    def rank(t):
        weight = float(w[t])
        if weight != weight:
            weight = float("-inf")
        safe = int(p[t]) + recent >= following or int(p[t]) < sinks
        return (not safe, -weight, t)

    kept = set(sorted(range(n), key=rank)[:m])
    freed = [t for t in range(m) if t not in kept]
    moved = sorted(t for t in kept if t >= m)
    source = list(range(m))
    for a, b in zip(freed, moved):
        source[a] = b
    return source, freed, moved
