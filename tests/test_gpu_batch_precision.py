"""How exact the decode attention over the paged cache is, against its definition in 64 bits: tighter than the worst-case
bounds of test_gpu_batch_ops.py, at the places where a term, a digit or a rounding sum could go missing unnoticed.

FP32 rows: the error over the norm of the output.  The softmax puts its weight on keys of a score of about the scores'
variance: 4 nats, 6 in log2 units, for queries of spread 2.  A score of z is off by some eight roundings of e |z|, a weight by
ln 2 times that and 4 e: 0.69 * 6 * 8 e + 4 e = 2.2e-6, and the sums add less: 3e-6.

16-bit rows: the share of outputs that are not the nearest value of their type.  What was computed is off by an error of r of the norm,
and a border between two values lies between it and the exact value for |error| / spacing of them: of the elements above a
quarter of the norm's share (1 / value averages 1.3 there) 0.8 * 1.3 * r / spacing, the spacing relative to the value 2^-7.5 (BF16) and 2^-10.5
(F16) on average.  F16 rows: a score is one tensor-core sum of up to 16 products that are cut off, each by up to 2 e of
the sum, 0.69 * 6 * 32 e = 7.9e-6 of a weight: r = 8e-6, a share of 1.2 %.  BF16 rows: weights of 11 bits, off by 2^-10 / sqrt(12) over
their leading digits' average of 1.44: r = 2e-4, a share of 3.8 %.  Twice that is allowed."""
import math

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from tests import batch_cache as bc  # noqa: E402
from tests.batch_cache import F16, Q4H, Q8, PagedCache, u32  # noqa: E402

E = 2.0 ** -24
F32, BF16, HF16 = torch.float32, torch.bfloat16, torch.float16
RELATIVE = {F32: 3e-6, HF16: 8e-6, BF16: 2e-4}
WRONG = {HF16: 0.024, BF16: 0.076}


def rand(shape, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda") * spread


def error(got, want):
    return float((got.double() - want).norm() / want.norm())


def wrongly_rounded(got, want):
    """The share of the elements that are not the nearest value of their type, small ones left out."""
    counts = want.abs() >= 0.25 * want.norm() / math.sqrt(want.numel())
    return float((got != want.to(got.dtype))[counts].double().mean())


def check(got, want, dtype, extra=0.0):
    """`extra`: a relative error beside the ones above."""
    if dtype == F32:
        assert error(got, want) <= RELATIVE[F32] + extra, error(got, want)
    else:
        assert wrongly_rounded(got, want) <= WRONG[dtype] * (1 + extra / RELATIVE[dtype]), wrongly_rounded(got, want)


CASES = [  # q, kv, hd, encoding, page
    (16, 4, 128, F16, 64), (8, 8, 64, F16, 16), (6, 2, 192, F16, 48), (12, 2, 256, F16, 64),
    (16, 4, 128, Q4H, 64), (8, 8, 64, Q4H, 16), (6, 2, 192, Q4H, 48), (12, 2, 256, Q4H, 64),
    (16, 4, 128, Q8, 64), (5, 5, 64, Q8, 16), (6, 2, 192, Q8, 48), (12, 3, 256, Q8, 64)]


@pytest.mark.parametrize("dtype", [F32, BF16, HF16])
@pytest.mark.parametrize("q,kv,hd,enc,page", CASES)
def test_attention_precision(q, kv, hd, enc, page, dtype):
    lengths = [1500, 90, 17]
    cache = PagedCache(len(lengths), -(-1500 // page), page, enc, kv, hd, seed=hd + enc)
    query = rand((len(lengths), q * hd), 7, 2.0).to(dtype)
    out = torch.zeros((len(lengths), q * hd), dtype=dtype, device="cuda")
    bc.decode_attention(cache, query, u32(lengths), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    want = torch.stack([bc.exact_attention(cache, s, n, query[s], q, hd ** -0.5)[0] for s, n in enumerate(lengths)])
    if dtype == F32:
        for s in range(len(lengths)):
            check(out[s].view(q, hd), want[s], dtype)
    else:
        check(out.view(-1, q, hd), want, dtype)


@pytest.mark.parametrize("q,kv,hd,enc,n,dtype", [(8, 1, 64, F16, 70001, F32), (5, 1, 128, Q4H, 40000, F32), (16, 4, 128, Q8, 33333, F32),
                                                 (8, 1, 128, F16, 50000, BF16), (12, 2, 256, F16, 20000, HF16)])
def test_attention_precision_of_a_long_sequence(q, kv, hd, enc, n, dtype):
    cache = PagedCache(1, n // 256 + 1, 256, enc, kv, hd, seed=3)
    query = rand((1, q * hd), 4, 2.0).to(dtype)
    out = torch.zeros((1, q * hd), dtype=dtype, device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    check(out[0].view(q, hd), bc.exact_attention(cache, 0, n, query[0], q, hd ** -0.5)[0], dtype)


@pytest.mark.parametrize("q,kv,hd,enc,page", CASES)
def test_a_missing_term_would_show(q, kv, hd, enc, page):
    """The same comparison with the loss planted in the definition: a query of one term (F16 cache) or two digits (quantised) less
    than the kernel's, or weights of one F16 term."""
    n = 1500
    cache = PagedCache(1, -(-n // page), page, enc, kv, hd, seed=hd + enc)
    query = rand((1, q * hd), 7, 2.0)
    want, p, _, _, _ = bc.exact_attention(cache, 0, n, query[0], q, hd ** -0.5)
    if enc == F16:
        less = query.half().float()
    else:
        unit = query.view(q, hd).abs().amax(-1, keepdim=True) / (127 * 256)
        less = ((query.view(q, hd) / unit).round() * unit).view(1, -1)
    got = bc.exact_attention(cache, 0, n, less[0], q, hd ** -0.5)[0]
    assert error(got.float(), want) > 3e-6
    group = q // kv
    _, values, _ = cache.values(0, n)
    w = (p * (2.0 ** 10 / p.amax(-1, keepdim=True))).half().double()
    got = torch.einsum("hgt,thd->hgd", (w * p.amax(-1, keepdim=True) / 2.0 ** 10).view(kv, group, n), values).reshape(q, hd)
    assert error(got.float(), want) > 3e-6
    assert wrongly_rounded(got.half(), want) > WRONG[HF16]


# F16 rows: behind more than 14 nats the output is below F16's normal values
@pytest.mark.parametrize("dtype,gap", [(t, g) for t in (F32, BF16, HF16) for g in (10.0, 14.0, 16.0, 20.0, 23.0, 40.0) if t != HF16 or g <= 14.0])
@pytest.mark.parametrize("n", [40, 2048])
def test_attention_behind_a_key_that_adds_nothing(dtype, gap, n):
    """An attention sink: one key scores `gap` nats above all others and its V is zero, so that the output is made of weights
    far below the largest.  An error of that key's score (8 e |z|) is one of every weight."""
    q, kv, hd, page = 8, 2, 128, 64
    cache = PagedCache(1, -(-n // page), page, F16, kv, hd, seed=5)
    both = cache.pool.view(HF16).view(-1, 2, page, kv, hd)
    if dtype == HF16:
        both[:, 1] *= 1024.0
    query = rand((1, q * hd), 4)
    query[0].view(q, hd)[:, 0] = 8.0
    both[:, 0, :, :, 0] = 0.0                                # dimension 0 carries the gap alone
    first = both[int(cache.index[0, 0])]
    first[0, 0] = 0.0
    first[0, 0, :, 0] = gap * hd ** 0.5 / 8.0
    first[1, 0] = 0.0
    query = query.to(dtype)
    out = torch.zeros((1, q * hd), dtype=dtype, device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    want = bc.exact_attention(cache, 0, n, query[0], q, hd ** -0.5)[0]
    check(out[0].view(q, hd), want, dtype, 8 * E * gap)


@pytest.mark.parametrize("enc", [Q4H, Q8])
@pytest.mark.parametrize("gap", [10.0, 16.0, 20.0])
def test_attention_behind_a_quantised_key_that_adds_nothing(enc, gap):
    """The same over quantised caches, whose V scale counts into the reference: the sink's is the smallest there is, 2^-24.  At 20 nats
    the others' weight times scale (at least 2^-6) is above 2^-11 of the sink's, to which two F16 terms hold 22 bits."""
    q, kv, hd, page, n = 8, 2, 128, 64, 2048
    cache = PagedCache(1, n // page, page, enc, kv, hd, seed=5)
    half, records, at = cache.bytes // 2, page * kv, int(cache.index[0, 0])
    pool = cache.pool.view(-1, 2, half)
    query = rand((1, q * hd), 4)
    query[0].view(q, hd)[:, 0] = 8.0
    codes = 127 if enc == Q8 else 7
    for h in range(kv):
        # dimension 0 carries the gap alone: zero for every other key, the largest code for the first one
        if enc == Q8:
            token_major = pool.view(-1, 2, page, kv, hd + 2)
            token_major[:, 0, :, h, 0] = 0
            token_major[at, :, 0, h, :hd] = 0
            token_major[at, 0, 0, h, 0] = codes
            scales = cache.pool.view(HF16).view(-1, 2, page, kv, hd // 2 + 1)[at, :, 0, h, hd // 2]
        else:
            nibbles = pool[:, :, :records * hd // 2].view(-1, 2, kv, page, hd // 2)
            nibbles[:, 0, h, :, 0] &= 0xF0
            nibbles[at, :, h, 0] = 0
            nibbles[at, 0, h, 0, 0] = codes
            scales = pool[:, :, records * hd // 2:].view(HF16).view(-1, 2, kv, page)[at, :, h, 0]
        scales[0] = gap * hd ** 0.5 / 8.0 / codes
        scales[1] = 2.0 ** -24
    out = torch.zeros((1, q * hd), device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    want = bc.exact_attention(cache, 0, n, query[0], q, hd ** -0.5)[0]
    check(out[0].view(q, hd), want, F32, 8 * E * gap)


@pytest.mark.parametrize("q,kv,hd,enc,dtype", [(8, 4, 64, Q8, HF16), (8, 1, 64, F16, HF16), (8, 1, 128, Q4H, HF16), (8, 4, 128, Q8, F32),
                                               (8, 1, 64, F16, F32), (8, 1, 64, Q4H, F32)])
def test_attention_of_long_items_that_no_block_shares(q, kv, hd, enc, dtype):
    """As many long sequences as there are blocks, and V of one sign: a sum that drops a part of a rounding with each tile would
    be off by their number.  All sequences share one sequence's pages, which are only read."""
    n, sequences, page = 65536, 800, 256
    cache = PagedCache(1, n // page, page, enc, kv, hd, seed=5)
    if enc == F16:
        both = cache.pool.view(HF16).view(-1, 2, page, kv, hd)
        both[:, 1] = (1.0 + 0.25 * both[:, 1].float()).half()
    else:
        m, half = cache.mine(), cache.bytes // 2
        if enc == Q8:
            m.view(-1, 2, page * kv, hd + 2)[:, 1, :, :hd] &= 0x3F
        else:
            m[:, half:half + page * kv * hd // 2] &= 0x77
    many = PagedCache.__new__(PagedCache)
    many.__dict__.update(cache.__dict__)
    many.sequences, many.tables = sequences, cache.tables.expand(sequences, -1).contiguous()
    query = rand((sequences, q * hd), 4, 0.05).to(dtype)
    out = torch.zeros((sequences, q * hd), dtype=dtype, device="cuda")
    bc.decode_attention(many, query, u32([n] * sequences), q, hd ** -0.5, out)
    torch.cuda.synchronize()
    for s in (0, 401, 799):
        want = bc.exact_attention(cache, 0, n, query[s], q, hd ** -0.5)[0]
        check(out[s].view(q, hd), want, dtype)


@pytest.mark.parametrize("enc", [Q4H, Q8])
@pytest.mark.parametrize("n", [40, 9000])
def test_an_infinite_scale_of_a_value_leaves_the_weights(enc, n):
    """V of one key is infinite: the output is not a number that counts, the weights of the keys are."""
    q, kv, hd, page = 4, 1, 128, 64
    cache = PagedCache(1, -(-n // page), page, enc, kv, hd, seed=5)
    query = rand((1, q * hd), 4, 2.0)
    want = bc.exact_attention(cache, 0, n, query[0], q, hd ** -0.5)[1].view(kv, q, n).sum(1)
    at, place, half, records = int(cache.index[0, 0]), 7, cache.bytes // 2, page * kv
    halves = cache.pool.view(HF16)
    halves[at, (half + place * (hd + 2) + hd) // 2 if enc == Q8 else (half + records * hd // 2) // 2 + place] = float("inf")
    out, weights = torch.zeros(1, q * hd, device="cuda"), torch.zeros(1, kv, cache.capacity, device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, hd ** -0.5, out, None, weights)
    torch.cuda.synchronize()
    assert not bool(out.isfinite().any())
    # a weight: the score's eight roundings of at most e |z| (the largest is below 16 nats), twice, and the sum's
    assert bool(((weights[0, :, :n].double() - want).abs() <= want * (2 * 8 * 16 * E + 8 * math.sqrt(n) * E) + 1e-37).all())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [40, 9000])
def test_keys_that_all_score_minus_infinity_give_zeros(dtype, n):
    """Whatever their V holds."""
    q, kv, hd, page = 4, 2, 64, 64
    cache = PagedCache(1, -(-n // page), page, F16, kv, hd, seed=5)
    both = cache.pool.view(HF16).view(-1, 2, page, kv, hd)
    both[:, 0, :, :, 3] = float("-inf")
    both[:, 1, ::3] = float("nan")
    query = rand((1, q * hd), 4).abs().add(0.1).to(dtype)
    out = torch.full((1, q * hd), 7.0, dtype=dtype, device="cuda")
    weights = torch.full((1, kv, cache.capacity), -3.0, device="cuda")
    bc.decode_attention(cache, query, u32([n]), q, 0.1, out, None, weights)
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((weights[0, :, :n] == 0).all())
