"""Refusals of the batched cache operators: every argument the host can see is checked before any CUDA
call, so these run without a GPU (the pointers are never read)."""
import ctypes

import pytest

from quantum_llm_b200 import lib as ql

INVALID = -4
BIG = 1 << 40


@pytest.fixture(scope="module")
def L():
    return ql.load()


def cache(**over):
    f = dict(page_tables=0x1000, layer_offset=0, sequences=3, pages_per_sequence=4, page_tokens=64, encoding=ql.KV_F16, kv_heads=2, head_dim=128)
    f.update(over)
    return ql.KvBatch(*f.values())


BAD_CACHES = [dict(sequences=0), dict(sequences=65536), dict(kv_heads=0), dict(head_dim=96), dict(head_dim=0), dict(head_dim=512),
              dict(page_tables=None), dict(page_tables=0x1004), dict(pages_per_sequence=0), dict(page_tokens=0), dict(page_tokens=24),
              dict(encoding=3), dict(layer_offset=8), dict(pages_per_sequence=1 << 25, page_tokens=64),
              dict(pages_per_sequence=1, page_tokens=1 << 22, kv_heads=4), dict(kv_heads=4097)]


def store(L, c=None, **over):
    f = dict(row_type=ql.ROW_BF16, qkv=0x100000, qkv_stride=8 * 128, rows=3, q_heads=4, rotary_dim=128, q_norm=0x2000, k_norm=0x3000,
             eps=1e-6, inv_freq=0x4000, positions=0x5000, row_sequence=0x6000, row_slot=0x7000, query=0x200000, query_stride=4 * 128,
             key=0x300000, key_stride=2 * 128, slot_positions=0x8000, slot_stride=256, stream=None)
    f.update(over)
    return L.qllm_k_qk_norm_rope_store(c or cache(), *f.values())


def attend(L, c=None, **over):
    f = dict(row_type=ql.ROW_BF16, query=0x100000, query_stride=4 * 128, lengths=0x2000, q_heads=4, scale=0.1, weights_in=0x400000,
             weights_out=0x500000, weights_stride=256, out=0x200000, out_stride=4 * 128, workspace=0x600000, workspace_bytes=BIG, stream=None)
    f.update(over)
    return L.qllm_k_decode_attention(c or cache(), *f.values())


def trim(L, c=None, **over):
    f = dict(lengths_in=0x2000, lengths_out=0x2100, next_positions=0x2200, budget=100, recent=10, sinks=4, weights_in=0x400000,
             weights_out=0x500000, positions_in=0x600000, positions_out=0x700000, stride=256, workspace=0x800000, workspace_bytes=BIG, stream=None)
    f.update(over)
    return L.qllm_k_kv_evict(c or cache(), *f.values())


@pytest.mark.parametrize("call", [store, attend, trim])
@pytest.mark.parametrize("bad", BAD_CACHES)
def test_caches_outside_the_contract(L, call, bad):
    assert call(L, cache(**bad)) == INVALID and L.qllm_last_error()


def test_null_cache(L):
    assert L.qllm_k_qk_norm_rope_store(None, 0, None, 0, 0, 0, 0, None, None, 0.0, *[None] * 5, 0, None, 0, None, 0, None) == INVALID
    assert L.qllm_k_decode_attention(None, 0, None, 0, None, 0, 0.0, None, None, 0, None, 0, None, 0, None) == INVALID
    assert L.qllm_k_kv_evict(None, None, None, None, 0, 0, 0, None, None, None, None, 0, None, 0, None) == INVALID
    assert L.qllm_k_decode_attention_workspace_bytes(None, 4, 1) == 0 and L.qllm_k_kv_evict_workspace_bytes(None, 4) == 0


@pytest.mark.parametrize("bad", [
    dict(row_type=3), dict(qkv=None), dict(qkv=0x100008), dict(qkv_stride=8 * 128 - 8), dict(qkv_stride=8 * 128 + 4), dict(rows=0), dict(q_heads=0),
    dict(rotary_dim=144), dict(rotary_dim=24), dict(q_norm=None), dict(k_norm=None), dict(eps=-1.0), dict(eps=float("nan")),
    dict(eps=float("inf")), dict(inv_freq=None), dict(positions=None), dict(row_sequence=None, rows=4), dict(query=None), dict(query=0x200002),
    dict(query_stride=4 * 128 - 8), dict(key=0x300002), dict(key_stride=128), dict(slot_stride=255), dict(row_slot=None),
    dict(query=0x100000, query_stride=4 * 128), dict(query=0x100010, query_stride=8 * 128), dict(key=0x100000, key_stride=8 * 128),
    dict(key=0x200000)])
def test_norm_rope_store(L, bad):
    assert store(L, **bad) == INVALID and L.qllm_last_error()


@pytest.mark.parametrize("bad", [
    dict(row_type=3), dict(query=None), dict(query=0x100008), dict(query_stride=4 * 128 - 8), dict(query_stride=4 * 128 + 4), dict(lengths=None),
    dict(q_heads=0), dict(q_heads=5), dict(scale=float("nan")), dict(scale=float("inf")), dict(weights_out=None), dict(weights_stride=255),
    dict(out=None), dict(out=0x200004), dict(out_stride=128), dict(out=0x100000), dict(out=0x100010), dict(workspace=None),
    dict(workspace=0x600004), dict(workspace_bytes=0), dict(weights_in=0x500010)])
def test_decode_attention(L, bad):
    assert attend(L, **bad) == INVALID and L.qllm_last_error()


@pytest.mark.parametrize("bad", [
    dict(lengths_in=None), dict(lengths_out=None), dict(lengths_out=0x2004), dict(next_positions=None), dict(next_positions=0x2104), dict(budget=0),
    dict(recent=97), dict(sinks=91), dict(recent=0xFFFFFFFF, sinks=5), dict(weights_in=None), dict(weights_out=None), dict(weights_out=0x400004),
    dict(positions_in=None), dict(positions_out=None), dict(positions_out=0x600004), dict(positions_in=0x500000), dict(positions_out=0x500000),
    dict(positions_out=0x400000), dict(stride=255), dict(workspace=None), dict(workspace=0x800008), dict(workspace_bytes=64)])
def test_kv_evict(L, bad):
    assert trim(L, **bad) == INVALID and L.qllm_last_error()


def test_strides_that_cannot_be_addressed(L):
    far = 1 << 56
    assert store(L, qkv_stride=far) == INVALID and store(L, query_stride=far) == INVALID and store(L, key_stride=far) == INVALID
    assert store(L, slot_stride=far) == INVALID and attend(L, query_stride=far) == INVALID and attend(L, out_stride=far) == INVALID
    assert attend(L, weights_stride=far) == INVALID and trim(L, stride=far) == INVALID
    # 60000 sequences of 65536 heads
    many = dict(sequences=60000, kv_heads=1, head_dim=64)
    assert attend(L, cache(**many), q_heads=65536, query_stride=65536 * 64, out_stride=65536 * 64, out=0x100000 + (1 << 52)) == INVALID


def test_valid_arguments_without_a_gpu_are_an_error(L):
    """The checks pass, and the first question to the device fails: no call works on the CPU instead."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for call in (store, attend, trim):
        assert call(L) < 0 and call(L) != INVALID and L.qllm_last_error()
    assert store(L, cache(page_tables=None, pages_per_sequence=0, page_tokens=0), row_slot=None, row_sequence=None, slot_positions=None) != INVALID


def test_workspace_sizes_grow_with_the_batch(L):
    small, large = cache(), cache(sequences=300, pages_per_sequence=64)
    for weights in (0, 1):
        a, b = (L.qllm_k_decode_attention_workspace_bytes(c, 4, weights) for c in (small, large))
        assert 0 < a <= b
    # a score per query head and slot is what the weights cannot do without
    assert L.qllm_k_decode_attention_workspace_bytes(large, 4, 1) >= 300 * 4 * 64 * 64 * 4
    assert L.qllm_k_kv_evict_workspace_bytes(small, 100) < L.qllm_k_kv_evict_workspace_bytes(large, 100)
    # sizes past 32 bits
    wide = cache(sequences=1024, pages_per_sequence=2048)
    assert L.qllm_k_decode_attention_workspace_bytes(wide, 16, 1) > 1024 * 16 * 2048 * 64 * 4 > 1 << 32
    assert ctypes.sizeof(ql.KvBatch) == 40


@pytest.mark.parametrize("bad", [dict(sequences=0), dict(sequences=65536), dict(kv_heads=0), dict(kv_heads=4097), dict(head_dim=0), dict(head_dim=96),
                                 dict(encoding=3), dict(pages_per_sequence=1 << 25, page_tokens=64)])
def test_no_workspace_for_a_cache_that_is_refused(L, bad):
    assert L.qllm_k_decode_attention_workspace_bytes(cache(**bad), 4, 1) == 0 and L.qllm_k_kv_evict_workspace_bytes(cache(**bad), 100) == 0
    assert L.qllm_k_decode_attention_workspace_bytes(cache(page_tables=None), 4, 1) > 0


@pytest.mark.parametrize("bad", [b for b in BAD_CACHES if "page_tables" not in b])
def test_no_workspace_for_any_cache_that_the_calls_refuse(L, bad):
    assert L.qllm_k_decode_attention_workspace_bytes(cache(**bad), 4, 1) == 0 and L.qllm_last_error()
    assert L.qllm_k_kv_evict_workspace_bytes(cache(**bad), 100) == 0 and L.qllm_last_error()


@pytest.mark.parametrize("q_heads,over", [(0, {}), (5, {}), (65538, {}), (65536, dict(sequences=60000, kv_heads=1))])
def test_no_workspace_for_query_heads_that_the_attention_refuses(L, q_heads, over):
    assert L.qllm_k_decode_attention_workspace_bytes(cache(**over), q_heads, 0) == 0 and L.qllm_last_error()


@pytest.mark.parametrize("call,name", [(store, n) for n in ("q_norm", "k_norm", "inv_freq", "positions", "row_sequence", "row_slot", "slot_positions")] +
                         [(attend, n) for n in ("lengths", "weights_in", "weights_out")] +
                         [(trim, n) for n in ("lengths_in", "lengths_out", "next_positions", "weights_in", "weights_out", "positions_in", "positions_out")])
def test_lists_off_a_word_boundary(L, call, name):
    assert call(L, **{name: 0x900002}) == INVALID and b"4-byte" in L.qllm_last_error()


SIDE_BY_SIDE = [
    # query and key rows as columns of one buffer; both behind the row in a wider buffer; key before query
    (store, dict(query=0x200000, query_stride=6 * 128, key=0x200000 + 8 * 128, key_stride=6 * 128)),
    (store, dict(qkv_stride=14 * 128, query=0x100000 + 16 * 128, query_stride=14 * 128, key=0x100000 + 24 * 128, key_stride=14 * 128)),
    (store, dict(query=0x200000 + 4 * 128, query_stride=6 * 128, key=0x200000, key_stride=6 * 128)),
    (attend, dict(query=0x100000, query_stride=8 * 128, out=0x100000 + 8 * 128, out_stride=8 * 128)),
    (attend, dict(weights_in=0x400000, weights_out=0x400000 + 256 * 4, weights_stride=512)),
    (trim, dict(weights_in=0x400000, weights_out=0x400000, positions_in=0x400000 + 256 * 4, positions_out=0x400000 + 256 * 4, stride=512))]
ONE_OVER_ANOTHER = [
    (store, dict(query=0x200000, query_stride=6 * 128, key=0x200000 + 8 * 128 - 16, key_stride=6 * 128)),
    (store, dict(query=0x200000, query_stride=6 * 128, key=0x200000 + 8 * 128 + 16, key_stride=6 * 128)),       # its end over the next row
    (store, dict(query=0x200000, query_stride=6 * 128, key=0x200000 + 8 * 128, key_stride=12 * 128)),
    (store, dict(qkv_stride=14 * 128, query=0x100000 + 16 * 128 - 16, query_stride=14 * 128)),
    (attend, dict(query=0x100000, query_stride=8 * 128, out=0x100000 + 8 * 128 + 16, out_stride=8 * 128)),
    (attend, dict(query=0x100000, query_stride=8 * 128, out=0x100000 - 8 * 128 - 16, out_stride=8 * 128)),
    (attend, dict(weights_in=0x400000, weights_out=0x400000 + 255 * 4, weights_stride=512)),
    (trim, dict(weights_in=0x400000, weights_out=0x400000, positions_in=0x400000 + 257 * 4, positions_out=0x400000 + 257 * 4, stride=512))]


@pytest.mark.parametrize("call,over", SIDE_BY_SIDE)
def test_columns_of_one_buffer_do_not_overlap(L, call, over):
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses that pass the checks; test_gpu_batch_paths.py has the calls on a GPU")
    assert call(L, **over) != INVALID


@pytest.mark.parametrize("call,over", ONE_OVER_ANOTHER)
def test_columns_that_overlap_are_refused(L, call, over):
    assert call(L, **over) == INVALID and b"overlap" in L.qllm_last_error()


def test_rows_without_norm_weights_are_taken(L):
    """Both null: no norm.  One alone is refused (test_norm_rope_store)."""
    import torch
    if torch.cuda.is_available():
        pytest.skip("made-up addresses that pass the checks; test_gpu_batch_paths.py has the call on a GPU")
    assert store(L, q_norm=None, k_norm=None) != INVALID
