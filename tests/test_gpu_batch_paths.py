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
