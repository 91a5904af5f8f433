"""GPU tests of the operators for batches of sequences over the paged cache, each against its definition in
64 bits: per-head norm + rotation + record store, decode attention with the weight of each key, eviction.

Tolerances count roundings.  u is half a step of the output's type relative to the value (2^-8 bf16, 2^-11
f16, 2^-24 f32); e = 2^-24 is FP32's.  Derivations stand at each comparison."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import batch_cache as bc  # noqa: E402
from tests.batch_cache import F16, HALF_STEP, Q4H, Q8, PagedCache, u32  # noqa: E402

E = 2.0 ** -24
F32, BF16, HF16 = torch.float32, torch.bfloat16, torch.float16
PAD = 0xFFFFFFFF


def rand(shape, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * spread


def inv_freq(rot, theta=1e6):
    half = rot // 2
    return torch.tensor([theta ** (-i / half) for i in range(half)] or [0.0], dtype=F32, device="cuda")


# ------------------------------------------------------------------ norm + rotation + store

def close_norm(got, want, size, dtype):
    """Sum of squares (at most 5 + 16 additions deep), mean, root, reciprocal, two products, cos and sin (2 ulp and
    the angle's 2^-23 pi), two products and a sum of the rotation: fewer than 48 roundings, each at most e of the
    magnitudes `size` that the rotation adds up; then one rounding to the type (F16 below 2^-14: half a step is 2^-25)."""
    bound = HALF_STEP[dtype] * want.abs() + 48 * E * size + (2.0 ** -25 if dtype == HF16 else 0.0)
    assert got.shape == want.shape and bool(((got.double() - want).abs() <= bound * 1.0001).all())


def check_record(cache, s, slot, h, key, key_size, value):
    """K within the roundings above and one to the record; V exactly what rounding the row's values gives."""
    k, v, _ = cache.values(s)
    parts = cache.parts(cache.mine()[cache.index[s]])
    if cache.enc == F16:
        close_norm(k[slot, h].half(), key, key_size, HF16)
        assert torch.equal(v[slot, h], value.half().double())
        return
    top = 7.0 if cache.enc == Q4H else 127.0
    for got, want, slack, part in ((k[slot, h], key, 48 * E * key_size, parts[0]), (v[slot, h], value.double(), torch.zeros_like(key), parts[1])):
        scale = part[1].reshape(cache.capacity, cache.kv)[slot, h].double()
        amax = float(want.abs().max())
        # the scale: amax / top, off by the slack and rounded to F16
        assert abs(float(scale) - max(amax / top, 2.0 ** -24)) <= (float(slack.max()) + amax * 2 ** -11) / top + 2.0 ** -25
        # the code: within half a step of value / scale (plus slack), except where it saturates at top
        inside = want.clamp(-top * scale, top * scale)
        assert bool(((got - inside).abs() <= scale * (0.5 + 4 * E * top) + slack).all())


NORM_CASES = [
    # q, kv, hd, rot, type, encoding, page
    (40, 8, 128, 128, BF16, F16, 256), (32, 4, 128, 128, HF16, Q8, 64), (12, 2, 256, 64, F32, Q4H, 16), (5, 1, 64, 64, BF16, Q4H, 48),
    (3, 3, 192, 96, F32, Q8, 32), (8, 8, 64, 0, HF16, F16, 16), (6, 2, 192, 192, BF16, F16, 16), (1, 1, 256, 256, HF16, Q4H, 64),
    (7, 1, 128, 16, F32, F16, 16), (16, 16, 64, 32, BF16, Q8, 16)]


@pytest.mark.parametrize("q,kv,hd,rot,dtype,enc,page", NORM_CASES)
@pytest.mark.parametrize("rows", [1, 2, 37])
def test_norm_rope_store(q, kv, hd, rot, dtype, enc, page, rows):
    sequences, pages = 3, 4
    cache = PagedCache(sequences, pages, page, enc, kv, hd, layers=2, layer=1, seed=rows)
    other = cache.pool[:, :cache.bytes].clone()
    before = cache.records()
    width = (q + 2 * kv) * hd
    x = rand((rows, width + 16), 1 + rows, 1.5).to(dtype)[:, :width]           # rows further apart than they are wide
    x[0, :hd] = 0                                                             # a query head and a value head of zeros
    x[0, width - hd:] = 0
    q_norm, k_norm = 1 + 0.3 * rand(hd, 5), 1 + 0.3 * rand(hd, 6)
    inv = inv_freq(rot)
    sequence = [(r * 7) % sequences for r in range(rows)]
    slot, position = [], []
    for r in range(rows):
        slot.append(PAD if r % 9 == 4 else (page - 1 + 5 * (r // sequences)) % cache.capacity)
        position.append([0, 1, 4095, 1_000_003, 4_000_000_000][r % 5] + r)
    query = torch.full((rows + 1, q * hd + 32), 7.0, dtype=dtype, device="cuda")[:, :q * hd]
    key = torch.full((rows + 1, kv * hd), 7.0, dtype=dtype, device="cuda")
    spots = torch.full((sequences, kv, cache.capacity + 3), -5, dtype=torch.int32, device="cuda")
    bc.norm_rope_store(cache, x, q, rot, q_norm, k_norm, inv, u32(position), u32(sequence), u32(slot), query, key, spots)
    torch.cuda.synchronize()
    wq, wk, size = bc.exact_norm_rope(x, q, kv, hd, rot, q_norm, k_norm, inv, position)
    live = [r for r in range(rows) if slot[r] != PAD]
    close_norm(query[live].reshape(len(live), q, hd), wq[live], size[live][:, :q], dtype)
    close_norm(key[live].view(len(live), kv, hd), wk[live], size[live][:, q:], dtype)
    left = [r for r in range(rows + 1) if r not in live]                       # padding, and the row behind the last
    assert bool((query[left] == 7).all()) and bool((key[left] == 7).all())
    values = x.view(rows, -1) if x.is_contiguous() else x.contiguous()
    values = values.view(rows, q + 2 * kv, hd)[:, q + kv:].float()
    touched = torch.zeros(sequences, cache.capacity, dtype=torch.bool, device="cuda")
    for r in live:
        for h in range(kv):
            check_record(cache, sequence[r], slot[r], h, wk[r, h], size[r, q + h], values[r, h])
        touched[sequence[r], slot[r]] = True
        assert spots[sequence[r], :, slot[r]].tolist() == [position[r] - (1 << 32) if position[r] >= 1 << 31 else position[r]] * kv
    assert torch.equal(cache.records()[~touched], before[~touched])            # nothing else in the cache moved,
    assert torch.equal(cache.pool[:, :cache.bytes], other)                      # nor the other layer of the pages,
    untouched = ~torch.cat((touched, torch.zeros(sequences, 3, dtype=torch.bool, device="cuda")), 1)
    assert bool((spots.transpose(1, 2)[untouched] == -5).all())                 # nor the positions of other slots


def test_norm_rope_store_in_place_and_without_a_cache():
    q, kv, hd, rows = 6, 2, 128, 11
    x = rand((rows, (q + 2 * kv) * hd), 3).to(BF16)
    w = 1 + 0.1 * rand(hd, 4)
    inv, positions = inv_freq(hd), list(range(100, 100 + rows))
    cache = PagedCache(rows, 1, 16, F16, kv, hd)
    query, key = torch.zeros(rows, q * hd, dtype=BF16, device="cuda"), torch.zeros(rows, kv * hd, dtype=BF16, device="cuda")
    before = cache.pool.clone()
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32(positions), None, None, query, key)
    assert torch.equal(cache.pool, before)
    both = x.clone()
    bc.norm_rope_store(cache, both, q, hd, w, w, inv, u32(positions), None, None, both, both[:, q * hd:(q + kv) * hd])
    assert torch.equal(both[:, :q * hd], query) and torch.equal(both[:, q * hd:(q + kv) * hd], key)
    assert torch.equal(both[:, (q + kv) * hd:], x[:, (q + kv) * hd:])
    # without row_sequence row r belongs to sequence r; the records are the key rows before their rounding
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32(positions), None, u32([r % 16 for r in range(rows)]), query)
    wq, wk, size = bc.exact_norm_rope(x, q, kv, hd, hd, w, w, inv, positions)
    for r in range(rows):
        close_norm(cache.values(r)[0][r % 16].half(), wk[r], size[r, q:], HF16)


def test_norm_rope_store_skips_what_lies_outside_the_cache():
    q, kv, hd = 2, 1, 64
    cache = PagedCache(2, 3, 16, Q8, kv, hd, absent=[(0, 1)])
    before = cache.pool.clone()
    rows = 4
    x = rand((rows, (q + 2 * kv) * hd), 3)
    w, inv = torch.ones(hd, device="cuda"), inv_freq(hd)
    query = torch.zeros(rows, q * hd, device="cuda")
    # a slot on an absent page, a slot behind the last page, a sequence that is not there, a far slot
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32([1, 2, 3, 4]), u32([0, 1, 2, 1]), u32([17, 48, 0, 0xFFFFFFFE]), query)
    assert torch.equal(cache.pool, before)
    wq, _, size = bc.exact_norm_rope(x, q, kv, hd, hd, w, w, inv, [1, 2, 3, 4])
    close_norm(query.view(rows, q, hd), wq, size[:, :q], F32)


def test_norm_rope_store_many_rows_and_infinities():
    """More rows than one wave of blocks; an infinite or NaN value stays in its own head."""
    q, kv, hd, rows = 4, 2, 128, 3001
    x = rand((rows, (q + 2 * kv) * hd), 8).to(HF16)
    x[5, 3] = float("inf")
    x[6, q * hd] = float("nan")
    x[7, (q + kv) * hd + 1] = float("nan")                 # a value head: code 0
    cache = PagedCache(1, rows // 64 + 1, 64, Q8, kv, hd)
    w, inv = 1 + 0.1 * rand(hd, 4), inv_freq(hd)
    query = torch.zeros(rows, q * hd, dtype=HF16, device="cuda")
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32(range(rows)), u32([0] * rows), u32(range(rows)), query)
    wq, wk, size = bc.exact_norm_rope(x, q, kv, hd, hd, w, w, inv, range(rows))
    good = [r for r in range(rows) if r not in (5,)]
    close_norm(query[good].view(len(good), q, hd), wq[good], size[good][:, :q], HF16)
    assert torch.equal(query[5].view(q, hd)[1:].isfinite(), torch.ones(q - 1, hd, dtype=torch.bool, device="cuda"))
    k, v, _ = cache.values(0)
    for r in (0, 1, 8, 1500, 3000):
        for h in range(kv):
            check_record(cache, 0, r, h, wk[r, h], size[r, q + h], x[r].view(-1, hd)[q + kv + h].float())
    assert float(v[7, 0, 1]) == 0.0 and bool(v[7, 0].isfinite().all()) and bool(k[6].isfinite().all())


def test_norm_rope_store_needs_no_pages_without_slots():
    """page_tables null and no page geometry: rows are normed and rotated, nothing is stored."""
    q, kv, hd, rows = 3, 1, 192, 5
    x = rand((rows, (q + 2 * kv) * hd), 3).to(BF16)
    w, inv = 1 + 0.1 * rand(hd, 4), inv_freq(64)
    query = torch.zeros(rows, q * hd, dtype=BF16, device="cuda")
    bare = bc.ql.KvBatch(None, 0, 1, 0, 0, 0, kv, hd)
    bc.ql.check(bc.ql.load().qllm_k_qk_norm_rope_store(
        bare, bc.ql.ROW_BF16, x.data_ptr(), x.stride(0), rows, q, 64, w.data_ptr(), w.data_ptr(), 1e-6, inv.data_ptr(),
        u32([9, 8, 7, 6, 5]).data_ptr(), None, None, query.data_ptr(), query.stride(0), None, 0, None, 0, bc.stream()))
    torch.cuda.synchronize()
    wq, _, size = bc.exact_norm_rope(x, q, kv, hd, 64, w, w, inv, [9, 8, 7, 6, 5])
    close_norm(query.view(rows, q, hd), wq, size[:, :q], BF16)


def test_memory_that_is_not_the_device_s_is_refused():
    """A page table (rows) in host memory: refused on the host, no kernel runs."""
    cache = PagedCache(2, 2, 16, F16, 1, 64)
    host = cache.descriptor()
    table = cache.tables.cpu()
    host.page_tables = table.data_ptr()
    L, n = bc.ql.load(), u32([5, 5])
    x = rand((2, 4 * 64), 1)
    out = torch.zeros(2, 128, device="cuda")
    ws = torch.zeros(1 << 24, dtype=torch.uint8, device="cuda")
    w, p = torch.zeros(2, 1, 32, device="cuda"), torch.zeros(2, 1, 32, dtype=torch.int32, device="cuda")
    assert L.qllm_k_decode_attention(host, 0, x.data_ptr(), 256, n.data_ptr(), 2, 0.1, None, None, 0, out.data_ptr(), 128, ws.data_ptr(),
                                     ws.numel(), bc.stream()) == -4
    assert L.qllm_k_kv_evict(host, n.data_ptr(), n.data_ptr(), u32([5, 5]).data_ptr(), 4, 0, 0, w.data_ptr(), w.data_ptr(), p.data_ptr(),
                             p.data_ptr(), 32, ws.data_ptr(), ws.numel(), bc.stream()) == -4
    y = x.cpu()
    assert L.qllm_k_qk_norm_rope_store(cache.descriptor(), 0, y.data_ptr(), 256, 2, 2, 0, out.data_ptr(), out.data_ptr(), 1e-6, None, n.data_ptr(),
                                       None, n.data_ptr(), out.data_ptr(), 128, None, 0, None, 0, bc.stream()) == -4
    assert b"current device" in L.qllm_last_error()
    torch.cuda.synchronize()


@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
def test_a_page_pointer_off_its_boundary_stands_for_no_page(enc):
    q, kv, hd, page = 4, 2, 64, 16
    cache = PagedCache(1, 3, page, enc, kv, hd, seed=2)
    cache.tables[0, 1] += 8
    pool = cache.pool.clone()
    x = rand((1, (q + 2 * kv) * hd), 3)
    w, inv = torch.ones(hd, device="cuda"), inv_freq(hd)
    query, out = torch.zeros(1, q * hd, device="cuda"), torch.zeros(1, q * hd, device="cuda")
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32([20]), u32([0]), u32([20]), query)
    weights = torch.full((1, kv, 48), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32([40]), q, 0.2, out, None, weights)
    cache.tables[0, 1] = 0                         # what the oracle takes for absent
    check_attention(cache, query, [40], q, 0.2, out, None, weights, F32)
    cache.tables[0, 1] = cache.tables[0, 0] + 4
    scores, positions, n = rand((1, kv, 48), 4).exp(), torch.arange(48, device="cuda", dtype=torch.int32).expand(1, kv, 48).clone(), u32([16])
    bc.evict(cache, n, n, u32([16]), 16, 4, 0, scores, scores, positions, positions)
    torch.cuda.synchronize()
    assert torch.equal(pool, cache.pool)


# ------------------------------------------------------------------------------- attention

def attention_bounds(dtype, n, hd, p, spread, size, want, v_sum):
    """z = scale * q.K is off by d = size * (hd + 8) e: hd additions of products (exact or rounded once), the query
    held in at least 22 bits.  exp2 and its argument's rounding add 8 e (1 + |z|), |z| <= size.  A weight of p is off by
    twice that (itself and the sum it is divided by), and the sums over n keys by 8 sqrt(n) e (a random walk of n
    roundings, taken eight times).  Before it meets V a weight becomes one F16 term with 16-bit rows (half a step: 2^-11) and
    two with FP32 rows (2^-22).  F16's smallest step is 2^-24, and the weights are scaled so that the largest (times V's scale) is at
    least 2^7: whatever its size, a weight is off by up to 2^-25 / 2^7 = 2^-32 of the largest, which meets sum |V|; a quantised V's
    scales, which the largest includes, differ by less than 2^4 here."""
    rel = 2 * (size * (hd + 8) + 8 * (1 + size)) * E + 8 * math.sqrt(n + 1) * E
    weight = rel + (2.0 ** -22 if dtype == F32 else 2.0 ** -11)
    largest = p.amax(-1) if n else torch.zeros_like(size)
    out = HALF_STEP[dtype] * want.abs() + weight[:, None] * spread * 1.01 + 2.0 ** -28 * largest[:, None] * v_sum
    return out + (2.0 ** -25 if dtype == HF16 else 1e-37), rel


def check_attention(cache, query, lengths, q_heads, scale, out, weights_in, weights_out, dtype):
    group = q_heads // cache.kv
    for s, n in enumerate(lengths):
        n = min(n, cache.capacity)
        want, p, spread, size, v_sum = bc.exact_attention(cache, s, n, query[s], q_heads, scale)
        got = out[s].view(q_heads, cache.hd).double()
        bound, rel = attention_bounds(dtype, n, cache.hd, p, spread, size, want, v_sum)
        assert bool(got.isfinite().all()), f"sequence {s} of {n}"
        worst = ((got - want).abs() / bound).max()
        assert float(worst) <= 1.0, f"sequence {s} of {n}: {float(worst)} of the bound"
        if weights_out is None:
            continue
        total = p.view(cache.kv, group, n).sum(1)
        start = weights_in[s, :, :n].double() if weights_in is not None else torch.zeros_like(total)
        slack = (p * rel[:, None]).view(cache.kv, group, n).sum(1) + (group + 2) * E * (total + start.abs())
        assert bool(((weights_out[s, :, :n].double() - start - total).abs() <= slack + 1e-37).all()), f"weights of sequence {s} of {n}"
        assert bool((weights_out[s, :, n:] == -3).all())     # at and behind the length: left alone


LENGTHS = [0, 1, 2, 15, 16, 17, 63, 64, 65, 100, 127, 128, 129, 255, 256, 257, 500, 767, 768]
ATTENTION_CASES = [
    # q, kv, hd, type, encoding, page
    (40, 8, 128, BF16, F16, 256), (40, 8, 128, BF16, Q4H, 256), (40, 8, 128, HF16, Q8, 256), (32, 4, 128, HF16, F16, 64),
    (16, 16, 64, F32, F16, 16), (4, 2, 64, BF16, Q8, 48), (6, 1, 64, HF16, Q4H, 16), (12, 2, 256, F32, Q4H, 64),
    (12, 1, 128, BF16, F16, 48), (16, 1, 256, HF16, F16, 16), (24, 1, 192, F32, Q8, 96), (3, 1, 192, BF16, Q4H, 32), (5, 5, 256, BF16, Q8, 16),
    (17, 1, 128, F32, F16, 256), (8, 1, 128, F32, Q4H, 16), (10, 5, 64, F32, Q8, 768), (9, 3, 192, HF16, F16, 48), (6, 6, 192, F32, Q4H, 16),
    (8, 2, 192, F32, Q8, 16), (4, 4, 256, BF16, Q8, 48), (6, 3, 128, HF16, Q8, 32)]   # Q8 records: even and odd numbers of heads


@pytest.mark.parametrize("q,kv,hd,dtype,enc,page", ATTENTION_CASES)
@pytest.mark.parametrize("weights", ["none", "fresh", "added"])
def test_attention(q, kv, hd, dtype, enc, page, weights):
    cache = PagedCache(len(LENGTHS), 768 // page, page, enc, kv, hd, layers=2, layer=1, seed=q)
    n = len(LENGTHS)
    query = rand((n, q * hd + 16), 9, 2.0).to(dtype)[:, :q * hd]
    out = torch.full((n + 1, q * hd + 32), 7.0, dtype=dtype, device="cuda")[:, :q * hd]
    w_in = torch.rand(n, kv, 800, device="cuda") if weights == "added" else None
    w_out = torch.full((n, kv, 800), -3.0, device="cuda") if weights != "none" else None
    pool = cache.pool.clone()
    keep = bc.decode_attention(cache, query, u32(LENGTHS), q, hd ** -0.5, out, w_in, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, LENGTHS, q, hd ** -0.5, out, w_in, w_out, dtype)
    assert bool((out[n] == 7).all()) and torch.equal(pool, cache.pool) and keep is not None
    assert bool((out[0] == 0).all())
    # the same bits again, and in place
    again = torch.zeros_like(out)
    w_again = w_in.clone() if w_in is not None else None
    bc.decode_attention(cache, query, u32(LENGTHS), q, hd ** -0.5, again, w_again, w_again)
    torch.cuda.synchronize()
    assert torch.equal(again[:n], out[:n])
    if w_in is not None:
        for s, length in enumerate(LENGTHS):
            assert torch.equal(w_again[s, :, :length], w_out[s, :, :length]) and torch.equal(w_again[s, :, length:], w_in[s, :, length:])


@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_attention_ignores_what_lies_behind_the_length(enc, dtype):
    """NaN and infinities in the rest of the last tile, absent pages inside, a length beyond the capacity."""
    q, kv, hd, page = 8, 2, 128, 32
    lengths = [1, 31, 33, 70, 96, 4_000_000_000, 64]
    absent = [(3, 1), (5, 0), (6, 0), (6, 1)]
    cache = PagedCache(len(lengths), 3, page, enc, kv, hd, absent=absent, seed=4)
    for s, n in enumerate(lengths):
        for p in range(3):
            tail = cache.mine()[int(cache.index[s, p])]
            (k, ks), (v, vs) = cache.parts(tail[None])
            for codes, scales in ((k, ks), (v, vs)):
                bad = torch.arange(page, device="cuda") + p * page >= n
                if scales is not None:
                    scales[:, bad] = float("nan")
                else:
                    codes[:, bad] = float("inf")
            # write the parts back in their layout
            flat = []
            for codes, scales in ((k, ks), (v, vs)):
                if enc == F16:
                    flat.append(bc.raw(codes).reshape(-1))
                elif enc == Q8:
                    flat.append(torch.cat((bc.raw(codes), bc.raw(scales[..., None])), -1).reshape(-1))
                else:
                    flat += [bc.raw(codes.transpose(1, 2)).reshape(-1), bc.raw(scales.transpose(1, 2)[..., None]).reshape(-1)]
            tail.copy_(torch.cat(flat))
        for p in [b for a, b in absent if a == s]:
            cache.mine()[int(cache.index[s, p])] = 0x7F        # nobody reads it
    query = rand((len(lengths), q * hd), 3).to(dtype)
    out = torch.full((len(lengths), q * hd), 7.0, dtype=dtype, device="cuda")
    w_out = torch.full((len(lengths), kv, 96), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, 0.3, out, None, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths, q, 0.3, out, None, w_out, dtype)
    assert bool((out[6] == 0).all()) and bool((w_out[6, :, :64] == 0).all())    # every slot absent


@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
@pytest.mark.parametrize("dtype", [F32, BF16, HF16])
@pytest.mark.parametrize("kind", ["peaked", "flat", "negative scale", "tiny", "huge", "growing"])
def test_attention_value_ranges(enc, dtype, kind):
    q, kv, hd, page, n = 5, 1, 128, 64, 700
    cache = PagedCache(1, 11, page, enc, kv, hd, seed=6)
    query = rand((1, q * hd), 5)
    scale = hd ** -0.5
    if kind == "peaked":
        query *= 8
    elif kind == "flat":
        query *= 0
    elif kind == "negative scale":
        scale = -scale
    elif kind == "tiny":                                       # scores and values far below 1, an F16 or scale near its smallest
        query *= 1e-3
        if enc == F16:
            cache.fill(torch.Generator(device="cuda").manual_seed(1), 2.0 ** -16)
        else:
            for codes, scales in cache_scales(cache):
                scales.fill_(2.0 ** -24)
    elif kind == "huge":                                       # query values that F16 does not hold, large keys
        query = query.clamp(-3, 3) * 2.0 ** (100 if dtype != HF16 else 12)
        scale = scale * 2.0 ** (-100 if dtype != HF16 else -12)
    elif kind == "growing":                                    # the running maximum grows with every tile
        query = query.abs() + 0.1
        if enc == F16:
            ramp = torch.linspace(-2, 2, cache.capacity, device="cuda").view(-1, page, 1, 1)
            both = cache.pool.view(HF16).view(-1, 2, page, kv, hd)
            both[cache.index[0], 0] = ramp.expand(-1, page, kv, hd).half()
    query = query.to(dtype)
    out = torch.zeros((1, q * hd), dtype=dtype, device="cuda")
    w_out = torch.full((1, kv, 704), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, scale, out, None, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, [n], q, scale, out, None, w_out, dtype)


def cache_scales(cache):
    """The scales of a quantised cache of one layer as writable views [pages of the pool, records]."""
    records = cache.page * cache.kv
    half = cache.bytes // 2
    for at in (0, half):
        b = cache.pool[:, at:at + half]
        if cache.enc == Q8:
            yield None, b.view(torch.float16).view(-1, records, cache.hd // 2 + 1)[:, :, -1] if cache.pool.shape[1] == half else \
                cache.pool.view(torch.float16).view(-1, 2, records, cache.hd // 2 + 1)[:, at // half, :, -1]
        else:
            yield None, cache.pool.view(torch.float16)[:, (at + records * cache.hd // 2) // 2:(at + half) // 2]


@pytest.mark.parametrize("q,kv,hd,enc,n,dtype", [(8, 1, 64, F16, 70001, BF16), (5, 1, 128, Q4H, 40000, F32), (16, 2, 128, Q8, 33333, HF16)])
def test_attention_long(q, kv, hd, enc, n, dtype):
    """One long sequence (split over the whole GPU) beside one of a single token."""
    page = 256
    cache = PagedCache(2, n // page + 1, page, enc, kv, hd, seed=2)
    query = rand((2, q * hd), 3, 2.0).to(dtype)
    out = torch.zeros((2, q * hd), dtype=dtype, device="cuda")
    w_out = torch.full((2, kv, cache.capacity), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32([1, n]), q, hd ** -0.5, out, None, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, [1, n], q, hd ** -0.5, out, None, w_out, dtype)
    # every query head's weights sum to one
    assert torch.allclose(w_out[1, :, :n].double().sum(-1), torch.full((kv,), float(q // kv), dtype=torch.float64, device="cuda"), rtol=1e-4)


@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
@pytest.mark.parametrize("dtype", [F32, BF16, HF16])
def test_attention_passes_nan_and_infinity_on(enc, dtype):
    """A NaN or an infinity in a query head makes that head NaN and its kv head's weights, nothing else; one in a key's record
    makes every head that reads it NaN.  One long sequence (joined parts) and one short one."""
    q, kv, hd, page, lengths = 8, 2, 128, 64, [9000, 40, 40]
    cache = PagedCache(3, 9000 // page + 1, page, enc, kv, hd, seed=6)
    query = rand((3, q * hd), 5).to(dtype)
    query[0, 1 * hd + 5] = float("nan")                  # head 1 of kv head 0
    query[1, 6 * hd + 7] = float("inf")                  # head 6 of kv head 1
    at = cache.index[2, 0]                              # sequence 2: key 13 of kv head 1
    if enc == F16:
        cache.pool.view(HF16).view(-1, 2, page, kv, hd)[at, 0, 13, 1, 3] = float("nan")
    else:
        record = 13 * kv + 1 if enc == Q8 else 1 * page + 13
        list(cache_scales(cache))[0][1][at, record] = float("nan")
    out = torch.zeros((3, q * hd), dtype=dtype, device="cuda")
    w_out = torch.full((3, kv, cache.capacity), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, 0.1, out, None, w_out)
    torch.cuda.synchronize()
    heads = out.view(3, q, hd)
    bad = torch.zeros(3, q, dtype=torch.bool, device="cuda")
    bad[0, 1] = bad[1, 6] = True
    bad[2, 4:] = True
    assert bool(heads[bad].isnan().all()) and bool(heads[~bad].isfinite().all())
    for s, h in ((0, 0), (1, 1), (2, 1)):
        assert bool(w_out[s, h, :lengths[s]].isnan().all()) and bool(w_out[s, 1 - h, :lengths[s]].isfinite().all())


def test_attention_many_short_sequences():
    """More sequences than blocks, none longer than two tiles, every third one empty."""
    sequences, q, kv, hd, page = 1500, 4, 2, 64, 16
    lengths = [0 if s % 3 == 0 else 1 + s % 40 for s in range(sequences)]
    cache = PagedCache(sequences, 3, page, F16, kv, hd, seed=2)
    query = rand((sequences, q * hd), 3).to(BF16)
    out = torch.full((sequences, q * hd), 7.0, dtype=BF16, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, 0.125, out)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths[:200], q, 0.125, out, None, None, BF16)
    assert bool((out[torch.tensor([n == 0 for n in lengths], device="cuda")] == 0).all())
    all_empty = torch.full((sequences, q * hd), 7.0, dtype=BF16, device="cuda")
    bc.decode_attention(cache, query, u32([0] * sequences), q, 0.125, all_empty)
    torch.cuda.synchronize()
    assert bool((all_empty == 0).all())


def test_attention_on_streams_and_in_a_graph():
    """Two streams at once with workspaces of their own; a captured call replayed after the lengths changed."""
    q, kv, hd, page = 8, 2, 128, 64
    cache = PagedCache(4, 8, page, Q8, kv, hd, seed=2)
    query = rand((4, q * hd), 3).to(HF16)
    length_sets = [[500, 3, 0, 64], [12, 512, 300, 1]]
    outs = [torch.zeros((4, q * hd), dtype=HF16, device="cuda") for _ in range(2)]
    spaces = [bc.attention_workspace(cache, q, True) for _ in range(2)]
    weights = [torch.full((4, kv, 512), -3.0, device="cuda") for _ in range(2)]
    lists = [u32(x) for x in length_sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                bc.decode_attention(cache, query, lists[i], q, 0.1, outs[i], None, weights[i], spaces[i])
    torch.cuda.synchronize()
    for i in range(2):
        check_attention(cache, query, length_sets[i], q, 0.1, outs[i], None, weights[i], HF16)
    out = torch.zeros_like(outs[0])
    now = lists[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        bc.decode_attention(cache, query, now, q, 0.1, out, None, None, spaces[0])
    for i in (0, 1, 0):
        now.copy_(lists[i])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, outs[i])


# -------------------------------------------------------------------------------- eviction

def evict_case(kind, sequences, kv, slots, lengths, seed):
    w = rand((sequences, kv, slots), seed).mul(2).exp()
    p = torch.arange(slots, device="cuda", dtype=torch.int32).expand(sequences, kv, slots).clone()
    if kind == "ties":
        w = (w * 2).round() / 2
    elif kind == "all equal":
        w = torch.ones_like(w)
    elif kind == "special":
        flat = w.view(-1)
        for i, x in enumerate((float("nan"), float("inf"), float("-inf"), 0.0, -0.0, -1.0, 1e-42)):
            flat[i::11] = x
    elif kind == "shuffled":
        for s, n in enumerate(lengths):
            for h in range(kv):
                p[s, h, :n] = torch.randperm(n, generator=torch.Generator().manual_seed(s * 31 + h)).int().cuda()
    elif kind == "same position":
        p.zero_()
    return w, p


@pytest.mark.parametrize("kind", ["plain", "ties", "all equal", "special", "shuffled", "same position"])
@pytest.mark.parametrize("enc,kv,hd,page", [(F16, 2, 128, 64), (Q4H, 3, 64, 48), (Q8, 1, 192, 16), (Q8, 2, 64, 96), (F16, 1, 256, 16)])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict(kind, enc, kv, hd, page, in_place):
    slots = -(-1100 // page) * page
    lengths = [0, 1, 64, 65, 199, 200, 201, 264, 399, 400, 401, 777, 1024, 1025, 1100]
    budget, recent, sinks = 200, 33, 4
    cache = PagedCache(len(lengths), slots // page, page, enc, kv, hd, layers=2, layer=1, seed=3)
    w, p = evict_case(kind, len(lengths), kv, slots, lengths, 11)
    following = [n if kind != "shuffled" else n + 7 for n in lengths]
    w_in, p_in, lengths_in = w.clone(), p.clone(), u32(lengths)
    w_out, p_out = (w_in, p_in) if in_place else (torch.full_like(w, -3), torch.full_like(p, -5))
    lengths_out = lengths_in if in_place else u32([77] * len(lengths))
    before, other = cache.records(), cache.pool[:, :cache.bytes].clone()
    keep = bc.evict(cache, lengths_in, lengths_out, u32(following), budget, recent, sinks, w_in, w_out, p_in, p_out)
    torch.cuda.synchronize()
    after = cache.records()
    assert lengths_out.tolist() == [min(n, budget) for n in lengths] and keep is not None
    assert torch.equal(other, cache.pool[:, :cache.bytes])
    w_cpu, p_cpu = w.cpu(), p.cpu()
    same = lambda a, b: torch.equal(a.contiguous().view(torch.int32), b.contiguous().view(torch.int32))  # noqa: E731
    for s, n in enumerate(lengths):
        m = min(n, budget)
        for h in range(kv):
            source, freed, moved = bc.exact_evict(w_cpu[s, h].tolist(), p_cpu[s, h].tolist(), n, following[s], budget, recent, sinks)
            at = torch.tensor(source, dtype=torch.long, device="cuda")
            assert same(w_out[s, h, :m], w[s, h][at]) and torch.equal(p_out[s, h, :m], p[s, h][at]), (s, h)
            assert bool((w_out[s, h, m:n] == 0).all())
            assert same(w_out[s, h, n:], w[s, h, n:] if in_place else torch.full_like(w[s, h, n:], -3))
            if not in_place:
                assert bool((p_out[s, h, m:] == -5).all())
            want = before[s, :, h].clone()
            want[:m] = before[s, at, h]
            assert torch.equal(after[s, :, h], want), (s, h)


@pytest.mark.parametrize("budget,recent,sinks", [(1, 0, 0), (1, 1, 0), (64, 64, 0), (64, 0, 64), (500, 100, 10), (4000, 0, 0), (5000, 10, 0), (0xFFFFFFFF, 5, 0)])
def test_evict_budgets(budget, recent, sinks):
    kv, hd, page, lengths = 2, 64, 16, [3333, 4096, 1]
    cache = PagedCache(3, 256, page, Q4H, kv, hd, seed=3)
    w, p = evict_case("ties", 3, kv, 4096, lengths, 5)
    w_out, p_out, n_out = torch.full_like(w, -3), torch.full_like(p, -5), u32([0] * 3)
    before = cache.records()
    bc.evict(cache, u32(lengths), n_out, u32(lengths), budget, recent, sinks, w, w_out, p, p_out)
    torch.cuda.synchronize()
    after = cache.records()
    for s, n in enumerate(lengths):
        m = min(n, budget)
        assert n_out.tolist()[s] == m
        for h in range(kv):
            source, _, _ = bc.exact_evict(w[s, h].tolist(), p[s, h].tolist(), n, n, budget, recent, sinks)
            at = torch.tensor(source, dtype=torch.long, device="cuda")
            assert torch.equal(w_out[s, h, :m], w[s, h][at]) and torch.equal(p_out[s, h, :m], p[s, h][at])
            assert torch.equal(after[s, :m, h], before[s, at, h])


@pytest.mark.parametrize("n,budget", [(70001, 30000), (131072, 131071), (50000, 49000)])
def test_evict_long(n, budget):
    """Rows longer than one block's shared memory holds, one with a length beyond the capacity."""
    kv, hd, page = 1, 64, 256
    cache = PagedCache(2, -(-n // page), page, Q4H, kv, hd, seed=3)
    slots = cache.capacity
    w, p = evict_case("ties", 2, kv, slots, [n, slots], 5)
    w_in, p_in = w.clone(), p.clone()
    lengths = u32([n, 3_000_000_000])
    before = cache.records()
    bc.evict(cache, lengths, lengths, u32([n, slots]), budget, 100, 4, w_in, w_in, p_in, p_in)
    torch.cuda.synchronize()
    after = cache.records()
    assert lengths.tolist() == [min(n, budget), min(slots, budget)]
    for s, full in enumerate((n, slots)):
        m = min(full, budget)
        source, _, _ = bc.exact_evict(w[s, 0].tolist(), p[s, 0].tolist(), full, full, budget, 100, 4)
        at = torch.tensor(source, dtype=torch.long, device="cuda")
        assert torch.equal(w_in[s, 0, :m], w[s, 0][at]) and torch.equal(p_in[s, 0, :m], p[s, 0][at])
        assert torch.equal(after[s, :m, 0], before[s, at, 0]) and bool((w_in[s, 0, m:full] == 0).all())


def test_evict_with_absent_pages():
    """Weights and positions move; a record whose page, or whose target's page, is absent does not."""
    kv, hd, page, n, budget = 1, 64, 16, 64, 20
    cache = PagedCache(1, 4, page, F16, kv, hd, absent=[(0, 3), (0, 1)], seed=3)
    w, p = evict_case("plain", 1, kv, 64, [n], 5)
    w_out, p_out, n_out = torch.zeros_like(w), torch.zeros_like(p), u32([0])
    before = cache.records()
    bc.evict(cache, u32([n]), n_out, u32([n]), budget, 5, 2, w, w_out, p, p_out)
    torch.cuda.synchronize()
    source, freed, moved = bc.exact_evict(w[0, 0].tolist(), p[0, 0].tolist(), n, n, budget, 5, 2)
    at = torch.tensor(source, dtype=torch.long, device="cuda")
    assert torch.equal(w_out[0, 0, :budget], w[0, 0][at]) and n_out.tolist() == [budget]
    want = before[0, :, 0].clone()
    for a, b in zip(freed, moved):
        if a // page not in (1, 3) and b // page not in (1, 3):
            want[a] = before[0, b, 0]
    assert torch.equal(cache.records()[0, :, 0], want)


def test_evict_on_two_streams():
    kv, hd, page, n, budget = 2, 64, 16, 2000, 700
    caches = [PagedCache(3, 128, page, Q8, kv, hd, seed=i) for i in range(2)]
    sets = [evict_case("plain", 3, kv, 2048, [n] * 3, 40 + i) for i in range(2)]
    spaces = [bc.evict_workspace(c, budget) for c in caches]
    outs = [(torch.zeros_like(w), torch.zeros_like(p), u32([0] * 3)) for w, p in sets]
    before, length = [c.records() for c in caches], u32([n] * 3)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        with torch.cuda.stream(streams[i]):
            bc.evict(caches[i], length, outs[i][2], length, budget, 50, 4, sets[i][0], outs[i][0], sets[i][1], outs[i][1], spaces[i])
    torch.cuda.synchronize()
    for i in range(2):
        after = caches[i].records()
        for s in range(3):
            for h in range(kv):
                source, _, _ = bc.exact_evict(sets[i][0][s, h].tolist(), sets[i][1][s, h].tolist(), n, n, budget, 50, 4)
                at = torch.tensor(source, dtype=torch.long, device="cuda")
                assert torch.equal(after[s, :budget, h], before[i][s, at, h]) and torch.equal(outs[i][1][s, h, :budget], sets[i][1][s, h][at])


# ------------------------------------------------------------------------------ a run together

@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("enc,dtype", [(F16, BF16), (Q8, F32), (Q4H, HF16)])
def test_streams_decoded_together_with_a_trimmed_cache(enc, dtype, graph):
    """Three streams decode a token a step: norm, rotation and record; attention that adds up the keys' weights;
    eviction once a stream is over its budget.  Every step is checked against the definitions over the cache as it then is."""
    sequences, q, kv, hd, page, budget, recent, sinks, steps = 3, 4, 2, 64, 16, 40, 8, 2, 60
    cache = PagedCache(sequences, 4, page, enc, kv, hd, seed=3)
    slots = cache.capacity
    norm, inv = 1 + 0.1 * rand(hd, 2), inv_freq(hd)
    lengths, following = u32([0, 30, 39]), u32([0, 30, 39])
    weights, positions = torch.zeros(sequences, kv, slots, device="cuda"), torch.zeros(sequences, kv, slots, dtype=torch.int32, device="cuda")
    for s, n in enumerate((0, 30, 39)):
        positions[s, :, :n] = torch.arange(n, device="cuda", dtype=torch.int32)
        weights[s, :, :n] = rand((kv, n), s).abs()
    qkv = torch.zeros(sequences, (q + 2 * kv) * hd, dtype=dtype, device="cuda")
    query, out = (torch.zeros(sequences, q * hd, dtype=dtype, device="cuda") for _ in range(2))
    space, trim = bc.attention_workspace(cache, q, True), bc.evict_workspace(cache, budget)

    def first():
        bc.norm_rope_store(cache, qkv, q, hd, norm, norm, inv, following, None, lengths, query, None, positions)
        lengths.add_(1)
        following.add_(1)

    def second():
        bc.decode_attention(cache, query, lengths, q, hd ** -0.5, out, weights, weights, space)

    def third():
        bc.evict(cache, lengths, lengths, following, budget, recent, sinks, weights, weights, positions, positions, trim)

    calls = [first, second, third]
    if graph:
        state = [t.clone() for t in (cache.pool, lengths, following, weights, positions)]
        graphs = []
        for call in calls:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                call()
            graphs.append(g)
        for t, kept in zip((cache.pool, lengths, following, weights, positions), state):
            t.copy_(kept)
        calls = [g.replay for g in graphs]
    for step in range(steps):
        qkv.copy_(rand(qkv.shape, 100 + step).to(dtype))
        n = [x + 1 for x in lengths.tolist()]
        where = following.tolist()
        calls[0]()
        torch.cuda.synchronize()
        assert lengths.tolist() == n
        wq, wk, size = bc.exact_norm_rope(qkv, q, kv, hd, hd, norm, norm, inv, where)
        close_norm(query.view(sequences, q, hd), wq, size[:, :q], dtype)
        for s in range(sequences):
            assert positions[s, :, n[s] - 1].tolist() == [where[s]] * kv
            check_record(cache, s, n[s] - 1, 0, wk[s, 0], size[s, q], qkv[s].view(-1, hd)[q + kv].float())
        held = weights.clone()
        for s in range(sequences):
            assert bool((held[s, :, n[s] - 1:] == 0).all())      # a new slot starts from nothing
        calls[1]()
        torch.cuda.synchronize()
        compare = weights.clone()
        for s in range(sequences):
            compare[s, :, n[s]:] = -3
        check_attention(cache, query, n, q, hd ** -0.5, out, held, compare, dtype)
        w, p, before = weights.clone(), positions.clone(), cache.records()
        calls[2]()
        torch.cuda.synchronize()
        assert lengths.tolist() == [min(x, budget) for x in n]
        for s in range(sequences):
            m = min(n[s], budget)
            for h in range(kv):
                source, _, _ = bc.exact_evict(w[s, h].tolist(), p[s, h].tolist(), n[s], where[s] + 1, budget, recent, sinks)
                at = torch.tensor(source, dtype=torch.long, device="cuda")
                assert torch.equal(weights[s, h, :m], w[s, h][at]) and torch.equal(positions[s, h, :m], p[s, h][at])
                assert torch.equal(cache.records()[s, :m, h], before[s, at, h])
                late = set(range(max(0, where[s] + 1 - recent), where[s] + 1)) | set(range(min(sinks, where[s] + 1)))
                assert late <= set(positions[s, h, :m].tolist())   # the last tokens and the sinks are always there
    assert following.tolist() == [steps, 30 + steps, 39 + steps]


@pytest.mark.parametrize("kind", ["ties", "same position"])
@pytest.mark.parametrize("in_place", [False, True])
def test_evict_rows_that_eight_blocks_do_not_hold(kind, in_place):
    """More slots than the shared memory of a whole cluster has room for: the keys are worked out again for every pass."""
    n, budget, hd, page = 400_007, 150_001, 64, 1024
    cache = PagedCache(1, -(-n // page), page, Q4H, 1, hd, seed=3)
    slots = cache.capacity
    w, p = evict_case("ties", 1, 1, slots, [n], 5)
    if kind == "same position":  # more protected slots than fit
        p = torch.where(torch.arange(slots, device="cuda") % 2 == 0, n - 1, p).int()
    w_in, p_in = w.clone(), p.clone()
    w_out, p_out = (w_in, p_in) if in_place else (torch.full_like(w, -3), torch.full_like(p, -5))
    lengths_out = u32([0])
    before = cache.records()
    bc.evict(cache, u32([n]), lengths_out, u32([n]), budget, 100, 4, w_in, w_out, p_in, p_out)
    torch.cuda.synchronize()
    after = cache.records()
    source, _, _ = bc.exact_evict(w[0, 0].tolist(), p[0, 0].tolist(), n, n, budget, 100, 4)
    at = torch.tensor(source, dtype=torch.long, device="cuda")
    assert lengths_out.tolist() == [budget]
    assert torch.equal(w_out[0, 0, :budget], w[0, 0][at]) and torch.equal(p_out[0, 0, :budget], p[0, 0][at])
    assert bool((w_out[0, 0, budget:n] == 0).all()) and torch.equal(after[0, :budget, 0], before[0, at, 0])
