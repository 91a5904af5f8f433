"""Paths of the batched cache operators that only some layouts and batch sizes take, each against its definition in 64 bits.
The bounds are those of test_gpu_batch_ops.py and test_gpu_batch_precision.py."""
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import batch_cache as bc  # noqa: E402
from tests.batch_cache import F16, Q4H, Q8, PagedCache, u32  # noqa: E402
from tests.test_gpu_batch_ops import check_attention, check_record, close_norm, inv_freq, rand  # noqa: E402

F32, BF16, HF16 = torch.float32, torch.bfloat16, torch.float16


# ------------------------------------------------------------------------- columns of one buffer

@pytest.mark.parametrize("dtype", [F32, BF16, HF16])
def test_queries_keys_and_outputs_as_columns_of_one_buffer(dtype):
    """Query and key rows side by side, then the attention's outputs beside the queries: the columns between are left alone."""
    q, kv, hd, rows, page = 6, 2, 128, 21, 16
    cache = PagedCache(rows, 2, page, F16, kv, hd, seed=3)
    x = rand((rows, (q + 2 * kv) * hd), 3).to(dtype)
    w, inv, positions = 1 + 0.1 * rand(hd, 4), inv_freq(hd), list(range(50, 50 + rows))
    gap = 32
    buffer = torch.full((rows, (2 * q + kv) * hd + 2 * gap), 7.0, dtype=dtype, device="cuda")
    query, key = buffer[:, :q * hd], buffer[:, q * hd + gap:(q + kv) * hd + gap]
    out = buffer[:, (q + kv) * hd + 2 * gap:]
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32(positions), None, u32([r % 20 for r in range(rows)]), query, key)
    torch.cuda.synchronize()
    wq, wk, size = bc.exact_norm_rope(x, q, kv, hd, hd, w, w, inv, positions)
    close_norm(query.reshape(rows, q, hd), wq, size[:, :q], dtype)
    close_norm(key.reshape(rows, kv, hd), wk, size[:, q:], dtype)
    assert bool((out == 7).all()) and bool((buffer[:, q * hd:q * hd + gap] == 7).all())
    before = buffer.clone()
    lengths = [1 + r % 32 for r in range(rows)]
    bc.decode_attention(cache, query, u32(lengths), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths, q, hd ** -0.5, out, None, None, dtype)
    assert torch.equal(buffer[:, :(q + kv) * hd + 2 * gap], before[:, :(q + kv) * hd + 2 * gap])


def test_weights_and_positions_as_columns_of_one_buffer():
    kv, hd, page, n, budget = 2, 64, 16, 60, 20
    cache = PagedCache(2, 4, page, Q8, kv, hd, seed=3)
    both = torch.zeros(2, kv, 2, 64, device="cuda")
    weights, positions = both[:, :, 0], both.view(torch.int32)[:, :, 1]
    weights.copy_(rand((2, kv, 64), 5).exp())
    positions.copy_(torch.arange(64, device="cuda", dtype=torch.int32).expand(2, kv, 64))
    w, p, before, lengths = weights.clone(), positions.clone(), cache.records(), u32([n, n - 30])
    bc.evict(cache, lengths, lengths, u32([n, n - 30]), budget, 5, 2, weights, weights, positions, positions)
    torch.cuda.synchronize()
    after = cache.records()
    for s, full in enumerate((n, n - 30)):
        m = min(full, budget)
        for h in range(kv):
            source, _, _ = bc.exact_evict(w[s, h].tolist(), p[s, h].tolist(), full, full, budget, 5, 2)
            at = torch.tensor(source, dtype=torch.long, device="cuda")
            assert torch.equal(weights[s, h, :m], w[s, h][at]) and torch.equal(positions[s, h, :m], p[s, h][at])
            assert torch.equal(after[s, :m, h], before[s, at, h]) and bool((weights[s, h, m:full] == 0).all())
            assert torch.equal(weights[s, h, full:], w[s, h, full:]) and torch.equal(positions[s, h, m:], p[s, h, m:])


# ------------------------------------------------------------------------- memory of the host

def test_lists_and_page_tables_of_the_host_are_refused():
    """Pageable host memory: refused before any launch.  Pinned lists are read as they are."""
    q, kv, hd = 4, 2, 64
    cache = PagedCache(2, 2, 16, F16, kv, hd, seed=3)
    host, table = cache.descriptor(), cache.tables.cpu()
    host.page_tables = table.data_ptr()
    L, n, kept, following = bc.ql.load(), u32([5, 20]), u32([0, 0]), u32([5, 20])
    far = n.cpu()
    pinned = far.pin_memory()
    x = rand((2, (q + 2 * kv) * hd), 1)
    query, out, ws = rand((2, q * hd), 2), torch.zeros(2, q * hd, device="cuda"), bc.attention_workspace(cache, q, False)
    w, p = torch.zeros(2, kv, 32, device="cuda"), torch.zeros(2, kv, 32, dtype=torch.int32, device="cuda")
    norm = torch.ones(hd, device="cuda")

    def store(descriptor, positions):
        return L.qllm_k_qk_norm_rope_store(descriptor, 0, x.data_ptr(), x.stride(0), 2, q, 0, norm.data_ptr(), norm.data_ptr(), 1e-6, None,
                                           positions.data_ptr(), None, n.data_ptr(), query.data_ptr(), q * hd, None, 0, None, 0, bc.stream())

    def attend(lengths):
        return L.qllm_k_decode_attention(cache.descriptor(), 0, query.data_ptr(), q * hd, lengths.data_ptr(), q, 0.1, None, None, 0,
                                         out.data_ptr(), q * hd, ws.data_ptr(), ws.numel(), bc.stream())

    def trim(lengths):
        return L.qllm_k_kv_evict(cache.descriptor(), lengths.data_ptr(), kept.data_ptr(), following.data_ptr(), 4, 0, 0, w.data_ptr(), w.data_ptr(),
                                 p.data_ptr(), p.data_ptr(), 32, ws.data_ptr(), ws.numel(), bc.stream())

    before = [t.clone() for t in (cache.pool, query, out, w, p, kept)]
    for refused in (store(host, n), store(cache.descriptor(), far), attend(far), trim(far)):
        assert refused == -4 and b"current device" in L.qllm_last_error()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.pool, query, out, w, p, kept)))
    assert attend(pinned) == 0
    torch.cuda.synchronize()
    check_attention(cache, query, [5, 20], q, 0.1, out, None, None, F32)


# ------------------------------------------------------------------------- models without a per-head norm

@pytest.mark.parametrize("q,kv,hd,rot,dtype,enc,page", [(40, 8, 128, 128, BF16, Q4H, 256), (32, 4, 128, 128, HF16, F16, 64), (12, 2, 256, 64, F32, Q8, 16),
                                                        (5, 1, 64, 0, BF16, F16, 48), (3, 3, 192, 96, F32, Q4H, 32)])
def test_rope_store_without_norm_weights(q, kv, hd, rot, dtype, enc, page):
    """q_norm and k_norm null: rotation and records of the rows as they are, whatever eps is; without a rotation the outputs are the inputs."""
    rows, sequences = 37, 3
    cache = PagedCache(sequences, 4, page, enc, kv, hd, layers=2, layer=1, seed=rows)
    x = rand((rows, (q + 2 * kv) * hd), 5, 1.5).to(dtype)
    x[3] = 0
    inv, position = inv_freq(rot), [[0, 1, 4095, 1_000_003, 4_000_000_000][r % 5] + r for r in range(rows)]
    sequence, slot = [r % sequences for r in range(rows)], [r // sequences for r in range(rows)]
    query, key = torch.zeros(rows, q * hd, dtype=dtype, device="cuda"), torch.zeros(rows, kv * hd, dtype=dtype, device="cuda")
    for eps in (0.0, 1e-6):
        bc.norm_rope_store(cache, x, q, rot, None, None, inv, u32(position), u32(sequence), u32(slot), query, key, eps=eps)
        torch.cuda.synchronize()
        heads = x.double().view(rows, q + 2 * kv, hd)[:, :q + kv]
        want, size, half = heads.clone(), heads.abs(), rot // 2
        if half:
            angle = torch.tensor([float(p) for p in position], dtype=torch.float64, device="cuda")[:, None, None] * inv.double()
            low, high = heads[..., :half], heads[..., half:rot]
            want[..., :half], want[..., half:rot] = low * angle.cos() - high * angle.sin(), high * angle.cos() + low * angle.sin()
            size[..., :half] = size[..., half:rot] = low.abs() + high.abs()
        else:
            assert torch.equal(query, x[:, :q * hd]) and torch.equal(key, x[:, q * hd:(q + kv) * hd])
        close_norm(query.view(rows, q, hd), want[:, :q], size[:, :q], dtype)
        close_norm(key.view(rows, kv, hd), want[:, q:], size[:, q:], dtype)
        values = x.view(rows, q + 2 * kv, hd)[:, q + kv:].float()
        for r in range(rows):
            for h in range(kv):
                check_record(cache, sequence[r], slot[r], h, want[r, q + h], size[r, q + h], values[r, h])


# ------------------------------------------------------------------------- the pages of the single-stream calls

@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_attention_reads_records_of_the_single_stream_store(enc, hd):
    """qllm_k_rope_kv_store writes two sequences' rows, one decode attention reads them."""
    q, kv, page, lengths = 4, 2, 64, [130, 61]
    cache = PagedCache(2, 3, page, enc, kv, hd, layers=2, layer=1, seed=3, fill=False)
    L, inv = bc.ql.load(), inv_freq(hd)
    top = {F16: 2.0 ** 11, Q4H: 7.0, Q8: 127.0}[enc]
    for s, n in enumerate(lengths):
        rows = rand((n, (q + 2 * kv) * hd), 10 + s)
        kept = rows.view(n, q + 2 * kv, hd)[:, q:].double()
        at = u32([0])
        bc.ql.check(L.qllm_k_rope_kv_store(rows.data_ptr(), n, q, kv, hd, 0, inv.data_ptr(), at.data_ptr(), 0, 0, cache.tables[s].data_ptr(),
                                           cache.layer * cache.bytes, page, enc, 0, bc.stream()))
        torch.cuda.synchronize()
        k, v, _ = cache.values(s, n)
        step = kept.abs().amax(-1, keepdim=True) / top      # a record is within a step of its row
        assert bool(((torch.cat((k, v), 1) - kept).abs() <= step).all())
    query = rand((2, q * hd), 5, 2.0)
    out, weights = torch.zeros(2, q * hd, device="cuda"), torch.full((2, kv, cache.capacity), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, hd ** -0.5, out, None, weights)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths, q, hd ** -0.5, out, None, weights, F32)


@pytest.mark.parametrize("enc", [F16, Q4H, Q8])
@pytest.mark.parametrize("hd", [64, 128])
def test_single_stream_attention_reads_records_of_the_batched_store(enc, hd):
    """qllm_k_qk_norm_rope_store writes two sequences' rows, qllm_k_attention reads each.  Its weights may be INT8 relative to the
    largest: off by 1 / 127 / sqrt(12) of it a key (each by itself), which meets a value of V's root mean square; four times the
    norm of that is allowed, and a BF16 step of the outputs."""
    q, kv, page, n = 4, 2, 64, 97
    cache = PagedCache(2, 2, page, enc, kv, hd, layers=2, layer=1, seed=3, fill=False)
    x = rand((2 * n, (q + 2 * kv) * hd), 3)
    w, inv = 1 + 0.1 * rand(hd, 4), inv_freq(hd)
    rows = torch.zeros(2 * n, q * hd, device="cuda")
    order = list(range(n))
    bc.norm_rope_store(cache, x, q, hd, w, w, inv, u32(order + order), u32([0] * n + [1] * n), u32(order + order), rows)
    L, split, splits = bc.ql.load(), 64, 3
    space = torch.empty(L.qllm_k_attention_workspace_bytes(1, q, hd, splits), dtype=torch.uint8, device="cuda")
    out, at = torch.zeros(1, q * hd, device="cuda"), u32([n - 1])
    for s in range(2):
        query = rows[s * n + n - 1:s * n + n].contiguous()
        bc.ql.check(L.qllm_k_attention(enc, cache.tables[s].data_ptr(), cache.layer * cache.bytes, page, query.data_ptr(), q * hd, 1, at.data_ptr(), 0,
                                       q, kv, hd, split, splits, 0, space.data_ptr(), out.data_ptr(), 0, bc.stream()))
        torch.cuda.synchronize()
        want, p, _, _, _ = bc.exact_attention(cache, s, n, query[0], q, hd ** -0.5)
        values = cache.values(s, n)[1]
        allowed = 4 * p.amax(-1) / 127 / 12 ** 0.5 * float(values.square().mean().sqrt()) * (n * hd) ** 0.5 + 2.0 ** -7 * want.norm(dim=-1)
        assert bool(((out.view(q, hd).double() - want).norm(dim=-1) <= allowed).all())
        # records read a slot further on would show
        wrong = torch.einsum("hgt,thd->hgd", p.view(kv, q // kv, n), values.roll(1, 0)).reshape(q, hd)
        assert bool(((wrong - want).norm(dim=-1) > allowed).all())


# ------------------------------------------------------------------------- batch sizes that choose another path

def blocks_of(cache, lengths, q_heads):
    """(items, items that more than one block of the attention's first launch works on), from its rule: equal shares of a line of 64-token
    units, an item's own cost before its tokens."""
    heads = 1 if cache.enc != Q8 else 4 if cache.kv % 4 == 0 else 2 if cache.kv % 2 == 0 else 1
    unit = 64 * heads * bc.layer_bytes(cache.enc, 1, 1, cache.hd)
    cost, tiles = -(-96 * 1024 // unit), -(-(q_heads // cache.kv) // 8)
    sizes = [-(-n // 64) + cost for n in lengths if n for _ in range(cache.kv // heads * tiles)]
    total = sum(sizes)
    per_sm = {64: 4, 128: 3}.get(cache.hd, 2)
    blocks = min(768, torch.cuda.get_device_properties(0).multi_processor_count * per_sm, total)
    at, split = 0, 0
    for n in sizes:
        first, last = at + cost, at + n - 1
        split += ((first + 1) * blocks - 1) // total != ((last + 1) * blocks - 1) // total
        at += n
    return len(sizes), split


@pytest.mark.parametrize("q,kv,hd,enc,dtype", [(32, 4, 64, F16, BF16), (32, 4, 128, F16, F32), (40, 8, 64, Q8, HF16), (24, 2, 192, Q4H, BF16), (24, 4, 256, Q8, F32)])
@pytest.mark.parametrize("weights", [False, True])
def test_attention_of_many_query_heads(q, kv, hd, enc, dtype, weights):
    """More than eight query heads to a multiprocessor, where one warp joins a head's parts instead of four, and items that blocks share."""
    sequences, page, top = 1300 // q + 14, 64, 3000
    lengths = [top, 0, 1] + [int(top * ((37 * s) % 101) / 101) + 200 for s in range(sequences - 4)] + [top - 1]
    lengths = [min(n, top) for n in lengths]
    cache = PagedCache(sequences, -(-top // page), page, enc, kv, hd, seed=3)
    assert sequences * q > 8 * torch.cuda.get_device_properties(0).multi_processor_count
    items, split = blocks_of(cache, lengths, q)
    assert split > items // 4
    query = rand((sequences, q * hd), 9, 2.0).to(dtype)
    out = torch.full((sequences, q * hd), 7.0, dtype=dtype, device="cuda")
    w_out = torch.full((sequences, kv, cache.capacity), -3.0, device="cuda") if weights else None
    bc.decode_attention(cache, query, u32(lengths), q, hd ** -0.5, out, None, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths, q, hd ** -0.5, out, None, w_out, dtype)
    assert bool((out[1] == 0).all())


@pytest.mark.parametrize("q,kv,enc,dtype", [(8, 8, F16, BF16), (48, 4, Q8, F32)])
def test_weights_of_many_rows(q, kv, enc, dtype):
    """More chunks of 512 tokens in a row than blocks that add up its weights (some 16 to a multiprocessor over all rows); the second
    case has more than eight query heads to a kv head, whose weights are added to the first ones'."""
    sequences, hd, page, top = 1280 // kv, 64, 64, 1700
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert -(-16 * sms // (sequences * kv)) < -(-top // 512)
    lengths = [(top * (s % 41)) // 40 for s in range(sequences)]
    cache = PagedCache(sequences, -(-top // page), page, enc, kv, hd, seed=3)
    query = rand((sequences, q * hd), 9, 2.0).to(dtype)
    out = torch.zeros((sequences, q * hd), dtype=dtype, device="cuda")
    w_in, w_out = torch.rand(sequences, kv, cache.capacity, device="cuda"), torch.full((sequences, kv, cache.capacity), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, hd ** -0.5, out, w_in, w_out)
    torch.cuda.synchronize()
    check_attention(cache, query, lengths, q, hd ** -0.5, out, w_in, w_out, dtype)


@pytest.mark.parametrize("dtype", [F32, BF16, HF16])
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("rot", [128, 32])
def test_norm_rope_store_of_many_passes(dtype, in_place, rot):
    """Rows enough for ten passes to a warp (2048 warps for 1500 rows of 56 heads, four to a pass): the values copied ahead wrap round."""
    q, kv, hd, rows, page = 40, 8, 128, 1500, 64
    assert (q + 2 * kv) // 4 * rows // 2048 >= 10
    cache = PagedCache(1, -(-rows // page), page, F16, kv, hd, seed=3)
    x = rand((rows, (q + 2 * kv) * hd), 8).to(dtype)
    given = x.clone()
    q_norm, k_norm, inv = 1 + 0.2 * rand(hd, 4), 1 + 0.2 * rand(hd, 5), inv_freq(rot)
    slot = list(range(rows))
    slot[7] = slot[900] = slot[rows - 1] = 0xFFFFFFFF
    if in_place:
        query, key = x, x[:, q * hd:(q + kv) * hd]
    else:
        query, key = torch.full((rows, q * hd), 7.0, dtype=dtype, device="cuda"), torch.full((rows, kv * hd), 7.0, dtype=dtype, device="cuda")
    before = cache.records()
    bc.norm_rope_store(cache, x, q, rot, q_norm, k_norm, inv, u32(range(rows)), u32([0] * rows), u32(slot), query, key)
    torch.cuda.synchronize()
    wq, wk, size = bc.exact_norm_rope(given, q, kv, hd, rot, q_norm, k_norm, inv, range(rows))
    live = torch.tensor([s != 0xFFFFFFFF for s in slot], device="cuda")
    close_norm(query[:, :q * hd].reshape(rows, q, hd)[live], wq[live], size[live][:, :q], dtype)
    close_norm(key.reshape(rows, kv, hd)[live], wk[live], size[live][:, q:], dtype)
    k, v, _ = cache.values(0, rows)
    close_norm(k[live].half(), wk[live], size[live][:, q:], HF16)
    assert torch.equal(v[live], given.view(rows, q + 2 * kv, hd)[live][:, q + kv:].half().double())
    assert torch.equal(cache.records()[0, :rows][~live], before[0, :rows][~live])
    if in_place:
        assert torch.equal(x[~live], given[~live]) and torch.equal(x[:, (q + kv) * hd:], given[:, (q + kv) * hd:])
    else:
        assert torch.equal(x, given) and bool((query[~live] == 7).all()) and bool((key[~live] == 7).all())


# ------------------------------------------------------------------------- several threads

def test_calls_from_several_threads():
    """Four threads, each with a stream, a cache and workspaces of its own, make the three calls at once; every thread's results are
    those of the same calls made alone."""
    import threading
    q, kv, hd, page, sequences, budget, steps = 8, 2, 128, 16, 3, 60, 25
    w, inv = 1 + 0.1 * rand(hd, 4), inv_freq(hd)

    def run(i):
        enc, dtype = (F16, Q4H, Q8, F16)[i], (BF16, HF16, F32, F32)[i]
        cache = PagedCache(sequences, 8, page, enc, kv, hd, seed=i)
        lengths, following = u32([50, 3, 59]), u32([50, 3, 59])
        weights = torch.zeros(sequences, kv, 128, device="cuda")
        positions = torch.arange(128, device="cuda", dtype=torch.int32).expand(sequences, kv, 128).clone()
        rows = [rand((sequences, (q + 2 * kv) * hd), 10 * i + s).to(dtype) for s in range(steps)]
        query = torch.zeros(sequences, q * hd, dtype=dtype, device="cuda")
        outs = torch.zeros(steps, sequences, q * hd, dtype=dtype, device="cuda")
        space, trim = bc.attention_workspace(cache, q, True), bc.evict_workspace(cache, budget)
        torch.cuda.synchronize()

        def go(barrier=None):
            with torch.cuda.stream(torch.cuda.Stream()):
                if barrier:
                    barrier.wait(30)
                for s in range(steps):
                    bc.norm_rope_store(cache, rows[s], q, hd, w, w, inv, following, None, lengths, query, None, positions)
                    lengths.add_(1)
                    following.add_(1)
                    bc.decode_attention(cache, query, lengths, q, hd ** -0.5, outs[s], weights, weights, space)
                    bc.evict(cache, lengths, lengths, following, budget, 8, 2, weights, weights, positions, positions, trim)
                torch.cuda.current_stream().synchronize()
        return go, (cache.pool, lengths, weights, positions, outs)

    alone = []
    for i in range(4):
        go, state = run(i)
        go()
        alone.append([t.clone() for t in state])
    calls, failed, barrier = [run(i) for i in range(4)], [], threading.Barrier(4)

    def work(go):
        try:
            go(barrier)
        except Exception as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(go,)) for go, _ in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    torch.cuda.synchronize()
    assert not failed and not any(t.is_alive() for t in threads)
    for (_, state), want in zip(calls, alone):
        assert all(torch.equal(bc.raw(a), bc.raw(b)) for a, b in zip(state, want))
