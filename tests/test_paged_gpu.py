"""The operators over a paged key-value cache against their definitions in 64 bits, with bounds from the arithmetic (paged_plain.py)."""
import random

import paged_plain
import pytest
import torch

from light_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


# ---------------------------------------------------------------- attention

def _cache(g, pages, KH, page, D, dtype, dev, layout="heads"):
    shape = {"heads": (pages, KH, page, D), "tokens": (pages, page, KH, D), "rows": (page, KH, pages, D)}[layout]
    order = {"heads": (0, 1, 2, 3), "tokens": (0, 2, 1, 3), "rows": (2, 1, 0, 3)}[layout]
    return torch.randn(shape, generator=g, device=dev).to(dtype).permute(order)


def _case(dev, dtype, lens, KH, G, D, page, seed=0, layout="heads", spare=2, width=0):
    """A batch over a shuffled pool; the rows that no sequence holds are NaN."""
    g = torch.Generator(dev).manual_seed(seed)
    held = [-(-n // page) for n in lens]
    pages, W = sum(held) + spare, max(max(held), 1) + width
    k, v = (_cache(g, pages, KH, page, D, dtype, dev, layout) for _ in range(2))
    perm = torch.randperm(pages, generator=g, device=dev).tolist()
    table = torch.full((len(lens), W), -7, dtype=torch.int32)
    used = torch.zeros((pages, page), dtype=torch.bool)
    for b, n in enumerate(lens):
        for w in range(held[b]):
            table[b, w] = perm.pop()
        for j in range(n):
            used[table[b, j // page], j % page] = True
    for c in (k, v):
        c.permute(0, 2, 1, 3)[~used.to(dev)] = float("nan")
    q = (2 * torch.randn((len(lens), KH * G, D), generator=g, device=dev)).to(dtype)
    return q, k, v, table.to(dev), torch.tensor(lens, dtype=torch.int32, device=dev)


def _check(q, k, v, table, lens, scale=None, window=0, softcap=0.0):
    scale = q.shape[2] ** -0.5 if scale is None else scale
    got = ops.PagedDecodeAttention(q, k, v, table, lens, scale, window=window, softcap=softcap)
    want, bound = paged_plain.attention(q, k, v, table, lens, scale, window, softcap)
    assert got.dtype == q.dtype and got.shape == q.shape and got.is_contiguous()
    off = (got.double() - want).abs()
    assert not torch.isnan(got).any(), (got.isnan().nonzero()[:4].tolist())
    assert bool((off <= bound).all()), (off / bound.clamp(min=1e-300)).max().item()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [16, 64, 80, 96, 128, 176, 256])
@pytest.mark.parametrize("G", [1, 4, 7, 8, 12])
def test_attention_heads_and_groups(cuda, dtype, D, G):
    _check(*_case(cuda, dtype, [1, 130, 0, 63, 400], 2, G, D, 16, seed=D + G))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("page", [1, 5, 8, 16, 48, 64, 100, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens", "rows"])
def test_attention_pages_and_layouts(cuda, dtype, page, layout):
    _check(*_case(cuda, dtype, [17, 300, 1, page, page + 1, max(page - 1, 1)], 3, 4, 64, page, seed=page, layout=layout))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4097])
def test_attention_one_sequence(cuda, dtype, n):
    _check(*_case(cuda, dtype, [n], 8, 4, 128, 16, seed=n))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 7, 64, 100, 1 << 30])
@pytest.mark.parametrize("softcap", [0.0, 0.01, 2.0, 50.0, 1e6])
def test_attention_window_and_cap(cuda, dtype, window, softcap):
    _check(*_case(cuda, dtype, [300, 5, 0, 64, 65, 1], 2, 5, 128, 24, seed=window % 97), window=window, softcap=softcap)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("KH,G", [(1, 16), (1, 20), (1, 71), (2, 33), (40, 1), (5, 3)])
def test_attention_group_sizes(cuda, dtype, KH, G):
    _check(*_case(cuda, dtype, [200, 3, 77], KH, G, 64, 16, seed=G))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B", [3, 40, 150, 1500])
def test_attention_ragged_batches(cuda, dtype, B):
    r = random.Random(B)
    lens = [int(2 ** r.uniform(0, 9)) * r.choice([0, 1, 1, 1]) for _ in range(B)]
    lens[B // 2] = 3000
    _check(*_case(cuda, dtype, lens, 2, 4, 64, 32, seed=B))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("KH,G,D,n", [(1, 1, 64, 30000), (1, 8, 128, 20011), (8, 4, 128, 9001), (2, 16, 256, 5000)])
def test_attention_long(cuda, dtype, KH, G, D, n):
    _check(*_case(cuda, dtype, [n], KH, G, D, 64, seed=n))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_large_scores(cuda, dtype):
    """One key takes all the weight, found late or early; scores of either sign in the hundreds."""
    q, k, v, table, lens = _case(cuda, dtype, [500, 500], 2, 4, 128, 16)
    for b, j in ((0, 3), (1, 477)):
        pg = table[b, j // 16]
        k[pg, :, j % 16] = q[b, ::4] * 4
    _check(q, k, v, table, lens, scale=0.5)
    _check(q, k, v, table, lens, scale=-0.5)
    _check(q, k, v, table, lens, scale=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_strided_query_and_shared_cache_tensor(cuda, dtype):
    q, k, v, table, lens = _case(cuda, dtype, [40, 129], 2, 4, 64, 16)
    wide = torch.zeros((2, 12, 64), dtype=dtype, device=cuda)
    wide[:, 2:10] = q
    both = torch.stack([k, v], 1)  # (pages, 2, KH, page, D)
    tables = torch.full((2, 50), -1, dtype=torch.int32, device=cuda)
    tables[:, 1:1 + table.shape[1]] = table
    want = _check(q, k, v, table, lens)
    got = ops.PagedDecodeAttention(wide[:, 2:10], both[:, 0], both[:, 1], tables[:, 1:1 + table.shape[1]], lens, 64 ** -0.5)
    assert torch.equal(got, want)
    off = torch.zeros((2, 8, 67), dtype=dtype, device=cuda)[..., 1:65]  # heads off 16 bytes
    off.copy_(q)
    assert torch.equal(ops.PagedDecodeAttention(off, k, v, table, lens, 64 ** -0.5), want)
    odd = q.transpose(1, 2).contiguous().transpose(1, 2)  # elements of a head apart
    assert torch.equal(ops.PagedDecodeAttention(odd, k, v, table.t().contiguous().t(), lens, 64 ** -0.5), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_rows_on_odd_addresses(cuda, dtype):
    q, k, v, table, lens = _case(cuda, dtype, [70, 5], 2, 3, 64, 16)
    k2, v2 = (torch.empty((*c.shape[:3], 67), dtype=dtype, device=cuda)[..., 1:65] for c in (k, v))
    k2.copy_(k), v2.copy_(v)
    _check(q, k2, v2, table, lens)
    q, k, v, table, lens = _case(cuda, dtype, [70, 5], 2, 3, 37, 16)
    _check(q, k, v, table, lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_infinities_and_nan(cuda, dtype):
    """What the formula gives: a key of score -inf weighs nothing, a NaN reaches its heads and no others; absent keys reach nobody."""
    q, k, v, table, lens = _case(cuda, dtype, [100, 100, 100], 2, 4, 64, 16)
    q.abs_()
    k[table[0, 1], :, 3] = float("-inf")
    v[table[1, 2], 1, 5] = float("nan")
    k[table[2], :, :] = float("-inf")
    got = ops.PagedDecodeAttention(q, k, v, table, lens, 0.125)
    clean = v.clone()
    clean[table[1, 2], 1, 5] = 0
    lengths = lens.clone()
    lengths[2] = 0
    want, bound = paged_plain.attention(q, k, clean, table, lengths, 0.125)
    assert got[1, 4:].isnan().all() and not got[1, :4].isnan().any()
    assert bool((got[2] == 0).all())  # nothing above -inf
    finite = paged_plain.attention(q, torch.where(k.isinf(), 0, k), clean, table, lengths, 0.125)[1]  # (the bound counts by the size of the scores)
    assert bool(((got.double() - want).abs()[0] <= finite[0]).all())
    assert bool(((got.double() - want).abs()[1, :4] <= bound[1, :4]).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [37, 128])
def test_attention_pages_and_lengths_outside(cuda, dtype, D):
    """Bad pages hold no keys, a length beyond the table stops at its end, a negative one is none; all of it is reported."""
    q, k, v, table, lens = _case(cuda, dtype, [90, 90, 90, 90, 33], 2, 4, D, 16)
    table[0, 2], table[1, 0], table[2, :] = -1, k.shape[0], 1 << 30
    lens[3], lens[4] = 5000, -3
    k[table[3].long(), :, :] = 0.5
    v[table[3].long(), :, :] = 0.25
    got = _check(q, k, v, table, lens)
    assert bool((got[2] == 0).all()) and bool((got[4] == 0).all())
    assert ops.paged_status(0) & 3 == 3


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_keys_and_values_in_different_orders(cuda, dtype):
    """Keys a page's head after the other, values a page's row after the other: their rows lie at different distances."""
    q, k, v, table, lens = _case(cuda, dtype, [200, 16, 333], 3, 4, 80, 16)
    v = v.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)
    _check(q, k, v, table, lens)
    _check(q, k, v, table, lens, window=50)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens", [[0, 0, 0], [1], [1] * 300, [5000] + [0] * 200 + [1], [16] * 40 + [3000] * 3 + [17] * 40, [0] * 130 + [700]])
def test_attention_batches_of_a_kind(cuda, dtype, lens):
    _check(*_case(cuda, dtype, lens, 2, 4, 64, 16, width=300))  # (a table much wider than the sequences)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_from_cold_memory_is_the_same_every_time(cuda, dtype):
    r = random.Random(4)
    case = _case(cuda, dtype, [int(2 ** r.uniform(0, 13)) for _ in range(40)], 4, 4, 128, 16)
    want = _check(*case)
    flush = torch.zeros(1 << 26, device=cuda)
    for _ in range(5):
        flush.add_(1)
        assert torch.equal(ops.PagedDecodeAttention(*case, 128 ** -0.5), want)


def test_attention_offsets_beyond_32_bits(cuda):
    """Pages 3 GB apart in one cache of 2^31 elements and more."""
    big = torch.zeros((1 << 31) + (1 << 22), dtype=torch.bfloat16, device=cuda)
    pages, KH, page, D = 3, 2, 16, 64
    c = big.as_strided((pages, KH, page, D), (1 << 30, page * D, D, 1))
    c.copy_(torch.randn((pages, KH, page, D), device=cuda))
    q = torch.randn((1, 4, D), device=cuda).to(torch.bfloat16)
    table, lens = torch.tensor([[2, 0, 1]], dtype=torch.int32, device=cuda), torch.tensor([41], dtype=torch.int32, device=cuda)
    _check(q, c, c, table, lens)
    k, v = torch.randn((5, 2, KH, D), device=cuda).to(torch.bfloat16)[:, 0], torch.randn((5, KH, D), device=cuda).to(torch.bfloat16)
    c2 = big.as_strided((pages, KH, page, D), (1 << 30, page * D, D, 1), 1 << 21)
    ops.QKNormRoPE(q.expand(5, 4, D), k, torch.zeros(5, dtype=torch.int64, device=cuda), torch.ones(D // 2, dtype=torch.float64, device=cuda), v=v, k_cache=c, v_cache=c2,
                   slots=torch.tensor([47, -1, -1, -1, -1], device=cuda))
    assert torch.equal(c[2, :, 15], k[0]) and torch.equal(c2[2, :, 15], v[0])
    del big


def test_attention_refusals(cuda):
    q, k, v, table, lens = _case(cuda, torch.bfloat16, [40, 20], 2, 4, 64, 16)
    call = ops.PagedDecodeAttention
    for bad in (lambda: call(q.double(), k, v, table, lens, 1.0), lambda: call(q[0], k, v, table, lens, 1.0), lambda: call(q.float(), k, v, table, lens, 1.0),
                lambda: call(q, k[..., :32], v, table, lens, 1.0), lambda: call(q[:, :3], k, v, table, lens, 1.0), lambda: call(q, k, v.float(), table, lens, 1.0),
                lambda: call(q, k, v, table.long(), lens, 1.0), lambda: call(q, k, v, table[:1], lens, 1.0), lambda: call(q, k, v, table, lens.long(), 1.0),
                lambda: call(q, k, v, table, lens[:1], 1.0), lambda: call(q, k, v, table, lens.cpu(), 1.0), lambda: call(q, k, v, table, lens, 1.0, window=-1),
                lambda: call(q, k, v, table, lens, 1.0, softcap=-1.0), lambda: call(q, k.transpose(2, 3).contiguous().transpose(2, 3), v, table, lens, 1.0),
                lambda: call(q, k.cpu(), v.cpu(), table, lens, 1.0), lambda: call(q, k, v, table[:, :0], lens, 1.0)):
        with pytest.raises(ValueError, match="PagedDecodeAttention"):
            bad()
    big = torch.zeros((2, 8, 320), dtype=torch.bfloat16, device=cuda)
    with pytest.raises(_lib.Light200Error, match="at most 256"):
        call(big, big.new_zeros((4, 2, 16, 320)), big.new_zeros((4, 2, 16, 320)), table, lens, 1.0)
    assert call(q[:0], k, v, table[:0], lens[:0], 1.0).shape == (0, 8, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rise", [0.02, 0.4, -0.02, -0.4])
@pytest.mark.parametrize("softcap", [0.0, 30.0])
def test_attention_scores_that_rise_or_fall(cuda, dtype, rise, softcap):
    """Every key's score a little above (below) the one before: a maximum that lags behind, never by more than it may."""
    q, k, v, table, lens = _case(cuda, dtype, [1000, 37], 2, 4, 64, 16)
    q.fill_(0.125)
    for b, n in enumerate((1000, 37)):
        for w in range(-(-n // 16)):
            k[table[b, w]] = ((torch.arange(16 * w, 16 * w + 16, device=cuda) - n / 2) * rise).to(dtype)[None, :, None]
    _check(q, k, v, table, lens, scale=0.125, softcap=softcap)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("softcap", [1e-20, 1e20])
def test_attention_caps_at_their_ends(cuda, dtype, softcap):
    _check(*_case(cuda, dtype, [1, 33, 700], 2, 4, 128, 16), softcap=softcap)


def test_attention_refuses_caps_that_overflow_and_extents_beyond_31_bits(cuda):
    q, k, v, table, lens = _case(cuda, torch.bfloat16, [40, 20], 2, 4, 64, 16)
    call = ops.PagedDecodeAttention
    for cap in (float("inf"), float("nan"), 3e38, 1e-38):
        with pytest.raises(ValueError, match="softcap"):
            call(q, k, v, table, lens, 1.0, softcap=cap)
    wide = k[:1, :1, :1].expand(1, 1, (1 << 32) + 16, 64)
    with pytest.raises(ValueError, match="2\\^31"):
        call(q, wide, wide, table, lens, 1.0)
    with pytest.raises(ValueError, match="2\\^31"):
        call(q, k, v, table[:, :1].expand(2, (1 << 32) + 3), lens, 1.0)
    with pytest.raises(ValueError, match="2\\^31"):
        call(q[:, :1].expand(2, (1 << 32) + 8, 64), k, v, table, lens, 1.0)
    pos, freq = torch.zeros(2, dtype=torch.int64, device=cuda), ops.RoPEFrequencies(64, 1e4)[0]
    with pytest.raises(ValueError, match="2\\^31"):
        ops.QKNormRoPE(q[:, :1].expand(2, (1 << 32) + 8, 64), q, pos, freq)


# ---------------------------------------------------------------- norm, rotation, cache rows

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D,R", [(128, 128), (64, 64), (128, 64), (80, 20), (96, 24), (256, 256), (256, 64), (40, 10), (8, 2), (7, 6), (112, 112)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("normed", [False, True])
def test_rotation(cuda, dtype, D, R, interleaved, normed):
    g = torch.Generator(cuda).manual_seed(D * R)
    T, NH, KH, page, pages = 37, 6, 2, 16, 5
    qkv = torch.randn((T, (NH + 2 * KH) * D), generator=g, device=cuda).to(dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((NH * D, KH * D, KH * D), 1))
    qw, kw = ((1 + 0.2 * torch.randn(D, generator=g, device=cuda)).to(dtype) for _ in range(2)) if normed else (None, None)
    freq, factor = ops.RoPEFrequencies(R, 10000.0, "yarn", 4.0, original=2048) if R > 2 else ops.RoPEFrequencies(R, 10000.0)
    positions = torch.randint(0, 1 << 20, (T,), generator=g, device=cuda)
    positions[0], positions[1] = 0, 131071
    slots = torch.randperm(pages * page, generator=g, device=cuda)[:T].contiguous()
    slots[-5:] = -1
    kc, vc = (torch.randn((pages, page, KH, D), generator=g, device=cuda).to(dtype).transpose(1, 2) for _ in range(2))
    kb, vb = kc.clone(), vc.clone()
    got, none = ops.QKNormRoPE(q, k, positions, freq, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved, factor=factor, v=v, k_cache=kc, v_cache=vc, slots=slots)
    assert none is None and got.shape == (T, NH, D) and got.dtype == dtype
    want, bound = paged_plain.rotated(q, qw, 1e-5, positions, freq, interleaved, factor)
    assert bool(((got.double() - want).abs() <= bound).all()), ((got.double() - want).abs() / bound).max().item()
    want, bound = paged_plain.rotated(k, kw, 1e-5, positions, freq, interleaved, factor)
    kept = slots[:-5]
    assert bool(((kc[kept // page, :, kept % page].double() - want[:-5]).abs() <= bound[:-5]).all())
    assert torch.equal(vc[kept // page, :, kept % page], v[:-5])
    others = torch.ones(pages * page, dtype=torch.bool, device=cuda)
    others[kept] = False
    rows = others.nonzero()[:, 0]
    assert torch.equal(kc[rows // page, :, rows % page], kb[rows // page, :, rows % page]) and torch.equal(vc[rows // page, :, rows % page], vb[rows // page, :, rows % page])
    # without a cache: the same keys, dense
    again, dense = ops.QKNormRoPE(q, k, positions, freq, q_weight=qw, k_weight=kw, eps=1e-5, interleaved=interleaved, factor=factor)
    assert torch.equal(again, got) and torch.equal(dense[:-5], kc[kept // page, :, kept % page])
    assert bool(((dense.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 2, 3, 64, 1000])
@pytest.mark.parametrize("NH,KH", [(1, 1), (32, 8), (28, 4), (71, 1)])
def test_rotation_sizes(cuda, dtype, T, NH, KH):
    g = torch.Generator(cuda).manual_seed(T)
    q, k = (torch.randn((T, n, 128), generator=g, device=cuda).to(dtype) for n in (NH, KH))
    w = torch.ones(128, dtype=dtype, device=cuda)
    positions = torch.arange(T, device=cuda) - 3  # negative ones turn back
    freq, _ = ops.RoPEFrequencies(128, 500000.0)
    gq, gk = ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=None)
    for x, got, weight in ((q, gq, w), (k, gk, None)):
        want, bound = paged_plain.rotated(x, weight, 1e-6, positions, freq, False, 1.0)
        assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,NH,KH,D", [(700, 32, 8, 128), (2000, 24, 8, 128), (5000, 32, 8, 128), (4000, 28, 4, 80), (3000, 16, 2, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_prompts_from_cold_memory(cuda, dtype, T, NH, KH, D, interleaved):
    """Many rounds of heads per warp, all of them from memory: what arrives late must be waited for."""
    g = torch.Generator(cuda).manual_seed(T)
    qkv = torch.randn((T, (NH + 2 * KH) * D), generator=g, device=cuda).to(dtype)
    q, k, v = (x.unflatten(1, (-1, D)) for x in qkv.split((NH * D, KH * D, KH * D), 1))
    w = (1 + 0.2 * torch.randn(D, generator=g, device=cuda)).to(dtype)
    freq, _ = ops.RoPEFrequencies(D, 500000.0)
    positions = torch.arange(T, device=cuda)
    pages = T // 16 + 1
    kc, vc = (torch.zeros((pages, KH, 16, D), dtype=dtype, device=cuda) for _ in range(2))
    slots = torch.randperm(pages * 16, generator=g, device=cuda)[:T].contiguous()
    flush = torch.zeros(1 << 26, device=cuda)
    for _ in range(3):
        flush.add_(1)
        got, _ = ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=w, interleaved=interleaved, v=v, k_cache=kc, v_cache=vc, slots=slots)
        want, bound = paged_plain.rotated(q, w, 1e-6, positions, freq, interleaved, 1.0)
        assert bool(((got.double() - want).abs() <= bound).all())
        want, bound = paged_plain.rotated(k, w, 1e-6, positions, freq, interleaved, 1.0)
        assert bool(((kc[slots // 16, :, slots % 16].double() - want).abs() <= bound).all())
        assert torch.equal(vc[slots // 16, :, slots % 16], v)
        kc.zero_(), vc.zero_()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotation_odd_addresses_and_orders(cuda, dtype):
    """Heads off 16 bytes, elements apart, one key for all tokens, weights in the middle of a tensor; a zero row stays zero."""
    g = torch.Generator(cuda).manual_seed(5)
    T, NH, KH, D = 9, 4, 2, 64
    base = torch.randn((T, NH + 1, D + 3), generator=g, device=cuda).to(dtype)
    q = base[:, 1:, 1:D + 1]
    q[3] = 0
    k = torch.randn((D, KH, 1), generator=g, device=cuda).to(dtype).permute(2, 1, 0).expand(T, KH, D)
    w = torch.randn(3 * D, generator=g, device=cuda).to(dtype)[1:2 * D + 1:2]
    positions, freq = torch.arange(2 * T, device=cuda)[::2], ops.RoPEFrequencies(D, 1e4)[0]
    gq, gk = ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=w)
    for x, got in ((q, gq), (k, gk)):
        want, bound = paged_plain.rotated(x, w, 1e-6, positions, freq, False, 1.0)
        assert bool(((got.double() - want).abs() <= bound).all())
    assert bool((gq[3] == 0).all())
    pages = torch.randn((3, KH, 16, D + 1), generator=g, device=cuda).to(dtype)
    kc, vc = pages[..., :D], pages.clone()[..., 1:]
    slots = torch.arange(T, device=cuda) * 5
    ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=w, v=k, k_cache=kc, v_cache=vc, slots=slots)
    assert torch.equal(kc[slots // 16, :, slots % 16], gk) and torch.equal(vc[slots // 16, :, slots % 16], k)


def test_rotation_slots_outside_are_reported_and_not_written(cuda):
    q, k = torch.randn((3, 4, 64), device=cuda), torch.randn((3, 2, 64), device=cuda)
    kc, vc = torch.zeros((2, 2, 8, 64), device=cuda), torch.zeros((2, 2, 8, 64), device=cuda)
    guard = kc.clone()
    freq = ops.RoPEFrequencies(64, 1e4)[0]
    ops.QKNormRoPE(q, k, torch.arange(3, device=cuda), freq, v=k, k_cache=kc, v_cache=vc, slots=torch.tensor([16, -1, 1 << 40], device=cuda))
    assert torch.equal(kc, guard) and torch.equal(vc, guard) and ops.paged_status(0) & 4


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [7, 64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_nothing(cuda, dtype, D, interleaved):
    """No frequencies: norm and the write of the rows alone.  No tokens: nothing."""
    g = torch.Generator(cuda).manual_seed(D)
    q, k, v = (torch.randn((19, n, D), generator=g, device=cuda).to(dtype) for n in (5, 2, 2))
    w = (1 + 0.2 * torch.randn(D, generator=g, device=cuda)).to(dtype)
    none, pos = torch.empty(0, dtype=torch.float64, device=cuda), torch.arange(19, device=cuda)
    kc, vc = (torch.zeros((2, 2, 16, D), dtype=dtype, device=cuda) for _ in range(2))
    got, _ = ops.QKNormRoPE(q, k, pos, none, q_weight=w, eps=1e-5, interleaved=interleaved, v=v, k_cache=kc, v_cache=vc, slots=pos)
    want, bound = paged_plain.rotated(q, w, 1e-5, pos, none, interleaved, 1.0)
    assert bool(((got.double() - want).abs() <= bound).all())
    assert torch.equal(kc.transpose(1, 2).reshape(32, 2, D)[:19], k) and torch.equal(vc.transpose(1, 2).reshape(32, 2, D)[:19], v)
    kb = kc.clone()
    got, _ = ops.QKNormRoPE(q[:0], k[:0], pos[:0], none, v=v[:0], k_cache=kc, v_cache=vc, slots=pos[:0])
    assert got.shape == (0, 5, D) and torch.equal(kc, kb)


def test_rotation_refusals(cuda):
    q, k = torch.zeros((3, 4, 64), device=cuda), torch.zeros((3, 2, 64), device=cuda)
    p, f, kc = torch.zeros(3, dtype=torch.int64, device=cuda), torch.ones(32, dtype=torch.float64, device=cuda), torch.zeros((2, 2, 8, 64), device=cuda)
    call = ops.QKNormRoPE
    for bad in (lambda: call(q.double(), k.double(), p, f), lambda: call(q, k.half(), p, f), lambda: call(q, k[:2], p, f), lambda: call(q[0], k, p, f), lambda: call(q, k, p.int(), f),
                lambda: call(q, k, p[:2], f), lambda: call(q, k, p, f.float()), lambda: call(q, k, p, torch.ones(33, dtype=torch.float64, device=cuda)), lambda: call(q, k, p, f.cpu()),
                lambda: call(q, k, p, f, q_weight=torch.ones(63, device=cuda)), lambda: call(q, k, p, f, k_weight=torch.ones(64, device=cuda).half()),
                lambda: call(q, k, p, f, v=k), lambda: call(q, k, p, f, v=k, k_cache=kc, v_cache=kc), lambda: call(q, k, p, f, v=q, k_cache=kc, v_cache=kc, slots=p),
                lambda: call(q, k, p, f, v=k, k_cache=kc.half(), v_cache=kc, slots=p), lambda: call(q, k, p, f, v=k, k_cache=kc[..., :32], v_cache=kc[..., :32], slots=p),
                lambda: call(q, k, p, f, v=k, k_cache=kc, v_cache=kc, slots=p.int()), lambda: call(q, k, p, f, v=k, k_cache=kc[:1].expand(2, 2, 8, 64), v_cache=kc, slots=p),
                lambda: call(q, k, p, f, v=k, k_cache=kc.transpose(2, 3).contiguous().transpose(2, 3), v_cache=kc, slots=p)):
        with pytest.raises(ValueError, match="QKNormRoPE"):
            bad()
    assert call(q[:0], k[:0], p[:0], f)[0].shape == (0, 4, 64)


# ---------------------------------------------------------------- pages

def _pool(B, page, width, longest, seed, spare):
    r = random.Random(seed)
    lens = [r.choice([0, 1, page, page * 2 - 1, r.randint(0, longest)]) for _ in range(B)]
    lens = [min(n, width * page) for n in lens]
    held = [-(-n // page) for n in lens]
    pages = list(range(sum(held) + spare))
    r.shuffle(pages)
    table = [[pages.pop() if w < h else -1 for w in range(width)] for h in held]
    return r, lens, table, pages + [-9] * (sum(held) + 3), len(pages)


def _t(x, dev, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=dev)


@pytest.mark.parametrize("B", [1, 2, 31, 300, 1024, 1025, 8192])
@pytest.mark.parametrize("page", [1, 16, 48])
@pytest.mark.parametrize("kind", ["decode", "prompts", "short of pages", "short of rows"])
@pytest.mark.parametrize("inplace", [False, True])
def test_advance(cuda, B, page, kind, inplace):
    width, longest = (12, 400) if page > 1 else (40, 30)
    r, lens, table, free, count = _pool(B, page, width, min(longest, width * page), B + page, 4 * B)
    if kind == "decode":
        new = [r.choice([0, 1, 1, 1]) for _ in range(B)]
    else:
        new = [r.randint(0, max(1, width * page - n + (2 if kind == "short of rows" else 0))) for n in lens]
    if kind == "short of pages":
        count = min(count, B)
    tokens = sum(new) + 3 if kind != "short of rows" else max(0, sum(new) * 2 // 3)
    T, L, N, F, K = _t(table, cuda), _t(lens, cuda), _t(new, cuda), _t(free, cuda), _t([count], cuda)
    want_table = [row[:] for row in table]
    pos, slot, starts, out, given, left = paged_plain.advance(want_table, lens, new, free, count, page, tokens)
    for _ in range(1 if inplace else 2):  # the same inputs once more: the same pages
        s = ops.PagedAdvance(T, L, N, F, K, page, tokens, inplace=inplace)
        assert s.positions.tolist() == pos and s.slots.tolist() == slot and s.starts.tolist() == starts
        assert s.lens.tolist() == out and s.granted.tolist() == given and s.free_count.tolist() == [left]
        assert T.tolist() == want_table and F.tolist() == free
    assert (s.lens is L and s.free_count is K) if inplace else (L.tolist() == lens and K.tolist() == [count])


@pytest.mark.parametrize("B", [1, 31, 300, 1025, 8192])
@pytest.mark.parametrize("page", [1, 16])
@pytest.mark.parametrize("share", [0.0, 0.1, 1.0])
@pytest.mark.parametrize("inplace", [False, True])
def test_release(cuda, B, page, share, inplace):
    r, lens, table, free, count = _pool(B, page, 12, 12 * page, B, 5)
    done = [r.random() < share for _ in range(B)]
    T, L, D, F, K = _t(table, cuda), _t(lens, cuda), _t(done, cuda, torch.bool), _t(free, cuda), _t([count], cuda)
    want_free = free[:]
    out, left = paged_plain.release(table, lens, done, want_free, count, page)
    for _ in range(1 if inplace else 2):
        n, c = ops.PagedRelease(T, L, D, F, K, page, inplace=inplace)
        assert n.tolist() == out and c.tolist() == [left] and F.tolist() == want_free and T.tolist() == table
    assert (n is L and c is K) if inplace else (L.tolist() == lens and K.tolist() == [count])


def test_pages_with_odd_counts_and_lengths(cuda):
    """Negative lengths count as none, a count of free pages outside the stack is cut to it, a full stack drops what it has no room for."""
    T, F = _t([[4, 5, -1], [6, -1, -1], [-1, -1, -1]], cuda), _t([0, 1, 2], cuda)
    s = ops.PagedAdvance(T, _t([17, -5, 3], cuda), _t([16, 4, -1], cuda), F, _t([99], cuda), 16, 21)
    assert s.lens.tolist() == [33, 4, 3] and s.granted.tolist() == [16, 4, 0] and s.free_count.tolist() == [1] and T.tolist() == [[4, 5, 2], [1, -1, -1], [-1, -1, -1]]
    assert s.positions.tolist() == list(range(17, 33)) + [0, 1, 2, 3, 0] and s.slots.tolist() == [5 * 16 + i for i in range(1, 16)] + [32, 16, 17, 18, 19, -1]
    assert ops.paged_status(0) & 8
    T, F = _t([[4, 5, 6], [7, 8, 9]], cuda), _t([0, 1, 2, 3], cuda)
    n, c = ops.PagedRelease(T, _t([48, 17], cuda), _t([1, 1], cuda, torch.bool), F, _t([-2], cuda), 16)
    assert n.tolist() == [0, 0] and c.tolist() == [4] and F.tolist() == [4, 5, 6, 7]
    n, c = ops.PagedRelease(T, _t([4800, 17], cuda), _t([1, 0], cuda, torch.bool), _t([0] * 9, cuda), _t([1], cuda), 16)
    assert n.tolist() == [0, 17] and c.tolist() == [4]


def test_release_reports_lengths_beyond_the_table(cuda):
    """(The bit stays set on the device: a child process has it clear.)"""
    import subprocess
    import sys

    from helpers import ROOT
    code = """
import torch
from light_b200 import ops
t = lambda x, d=torch.int32: torch.tensor(x, dtype=d, device="cuda")
T = t([[4, 5], [7, 8]])
for n, want in ((32, 0), (33, 8)):
    lens, count = ops.PagedRelease(T, t([n, 33]), t([1, 0], torch.bool), t([0] * 9), t([1]), 16)
    assert (lens.tolist(), count.tolist(), ops.paged_status(0)) == ([0, 33], [3], want), n
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT, timeout=300)


def test_advance_of_no_tokens_and_in_inference_mode(cuda):
    T, F = _t([[4, -1], [5, -1]], cuda), _t([0, 1, 2], cuda)
    s = ops.PagedAdvance(T, _t([16, 3], cuda), _t([0, 0], cuda), F, _t([3], cuda), 16, 0)
    assert s.positions.shape == s.slots.shape == (0,) and s.starts.tolist() == [0, 0, 0] and s.lens.tolist() == [16, 3] and s.free_count.tolist() == [3]
    with torch.inference_mode():
        s = ops.PagedAdvance(T, _t([16, 3], cuda), _t([1, 1], cuda), F, _t([3], cuda), 16, 2)
        s.slots.add_(0)
        lens, count = ops.PagedRelease(T, s.lens, _t([1, 0], cuda, torch.bool), F, s.free_count, 16)
    assert s.slots.is_inference() and s.slots.tolist() == [32, 5 * 16 + 3] and T.tolist() == [[4, 2], [5, -1]]
    assert lens.tolist() == [0, 4] and count.tolist() == [3] and F.tolist() == [0, 1, 4]  # (a stack of three: page 2 has no room)
    s = ops.PagedAdvance(T, lens, _t([0, 1], cuda), F, count, 16, 1)
    s.lens.add_(1)
    assert s.lens.tolist() == [1, 6] and s.granted.tolist() == [0, 1]


def test_advance_writes_rows_of_a_wider_table_only(cuda):
    wide = torch.full((3, 20), -5, dtype=torch.int32, device=cuda)
    s = ops.PagedAdvance(wide[:, 4:10], _t([0, 0, 0], cuda), _t([90, 1, 96], cuda), _t(list(range(40)), cuda), _t([40], cuda), 16, 187)
    assert s.granted.tolist() == [90, 1, 96] and bool((wide[:, :4] == -5).all()) and bool((wide[:, 10:] == -5).all()) and int((wide[:, 4:10] >= 0).sum()) == 13


def test_page_refusals(cuda):
    T, i, f = _t([[0, 1], [2, 3]], cuda), _t([1, 1], cuda), _t([4, 5], cuda)
    adv = lambda **k: ops.PagedAdvance(**{**dict(block_table=T, lens=i, new_lens=i, free_pages=f, free_count=f[:1], page_size=16, tokens=2), **k})  # noqa: E731
    rel = lambda **k: ops.PagedRelease(**{**dict(block_table=T, lens=i, done=i > 0, free_pages=f, free_count=f[:1], page_size=16), **k})  # noqa: E731
    for call, bad in [(adv, b) for b in (dict(new_lens=i[:1]), dict(new_lens=i.long()), dict(tokens=-1))] + [(rel, b) for b in (dict(done=i), dict(done=(i > 0)[:1]), dict(done=(i > 0).cpu()))] + \
            [(c, b) for c in (adv, rel) for b in (dict(block_table=T.long()), dict(block_table=T.t()), dict(block_table=T[:, :0]), dict(block_table=T[0]), dict(block_table=T[:1].expand(2, 2)),
                                                  dict(lens=i[:1]), dict(lens=i.long()), dict(lens=_t([1, 1, 1, 1], cuda)[::2]), dict(free_pages=f.long()), dict(free_pages=f[:0]),
                                                  dict(free_count=f), dict(page_size=0), dict(page_size=1 << 32), dict(lens=i.cpu()))]:
        with pytest.raises(ValueError, match="ops.Paged"):
            call(**bad)
    with pytest.raises(_lib.Light200Error, match="at most 8192"):
        adv(block_table=torch.zeros((8193, 1), dtype=torch.int32, device=cuda), lens=torch.zeros(8193, dtype=torch.int32, device=cuda), new_lens=torch.zeros(8193, dtype=torch.int32, device=cuda))
    assert adv().granted.tolist() == [1, 1]


# ---------------------------------------------------------------- together

class _Server:
    """A decode loop over one pool, and beside it every sequence's keys and values in a list of its own."""

    def __init__(self, dev, dtype, B, KH, G, D, page, width, pages, seed):
        self.dev, self.dtype, self.KH, self.G, self.D, self.page = dev, dtype, KH, G, D, page
        self.g = torch.Generator(dev).manual_seed(seed)
        self.table = torch.full((B, width), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(B, dtype=torch.int32, device=dev)
        self.free, self.count = torch.arange(pages, dtype=torch.int32, device=dev), _t([pages], dev)
        self.k, self.v = (torch.full((pages, KH, page, D), float("nan"), dtype=dtype, device=dev) for _ in range(2))
        self.freq, self.factor = ops.RoPEFrequencies(D, 10000.0)
        self.w = (1 + 0.1 * torch.randn(D, generator=self.g, device=dev)).to(dtype)

    def step(self, new, tokens, inputs=None):
        """One step; the last token of every request attends."""
        s = ops.PagedAdvance(self.table, self.lens, new, self.free, self.count, self.page, tokens, inplace=True)
        NH = self.KH * self.G
        qkv = inputs if inputs is not None else torch.randn((tokens, (NH + 2 * self.KH) * self.D), generator=self.g, device=self.dev).to(self.dtype)
        q, k, v = (x.unflatten(1, (-1, self.D)) for x in qkv.split((NH * self.D, self.KH * self.D, self.KH * self.D), 1))
        q, _ = ops.QKNormRoPE(q, k, s.positions, self.freq, q_weight=self.w, k_weight=self.w, factor=self.factor, v=v, k_cache=self.k, v_cache=self.v, slots=s.slots)
        last = (s.starts[1:] - 1).clamp(min=0)
        out = ops.PagedDecodeAttention(q[last], self.k, self.v, self.table, s.lens, self.D ** -0.5)
        return s, q, k, v, out, last


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_server_of_many_sequences(cuda, dtype):
    """Arrivals with prompts, decode steps, departures, pages used again: each sequence attends as if it were alone."""
    B, page = 7, 16
    s = _Server(cuda, dtype, B, 2, 4, 64, page, 20, 80, 1)
    r = random.Random(1)
    keys, values = [[] for _ in range(B)], [[] for _ in range(B)]
    for _ in range(25):
        new = [(r.choice([0, 0, r.randint(1, 100)]) if not keys[b] else r.choice([1, 1, 1, 0])) for b in range(B)]
        step, q, k, v, out, last = s.step(_t(new, cuda), sum(new) + 2)
        wk, bk = paged_plain.rotated(k, s.w, 1e-6, step.positions, s.freq, False, 1.0)
        granted, starts = step.granted.tolist(), step.starts.tolist()
        for b in range(B):
            for i in range(granted[b]):
                row = starts[b] + i
                slot = int(step.slots[row])
                kept = s.k[slot // page, :, slot % page]
                assert bool(((kept.double() - wk[row]).abs() <= bk[row]).all()) and torch.equal(s.v[slot // page, :, slot % page], v[row])
                keys[b].append(kept.clone())
                values[b].append(v[row])
            n = len(keys[b])
            assert n == int(step.lens[b])
            if n == 0:
                assert bool((out[b] == 0).all())
                continue
            # alone, in a cache of its own
            kk, vv = torch.stack(keys[b], 1)[None], torch.stack(values[b], 1)[None]  # (1, KH, n, D): one page
            want, bound = paged_plain.attention(q[last[b]][None], kk, vv, _t([[0]], cuda), _t([n], cuda), 64 ** -0.5)
            assert bool(((out[b].double() - want[0]).abs() <= bound[0]).all())
        done = [bool(keys[b]) and r.random() < 0.12 for b in range(B)]
        ops.PagedRelease(s.table, s.lens, _t(done, cuda, torch.bool), s.free, s.count, page, inplace=True)
        for b in range(B):
            if done[b]:
                keys[b], values[b] = [], []
        held = sum(-(-len(x) // page) for x in keys)
        assert int(s.count) + held == 80


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_is_the_step(cuda, dtype):
    """One decode step as a graph, replayed while the lengths grow past pages, against the same steps eagerly."""
    def fresh():
        s = _Server(cuda, dtype, 5, 2, 4, 128, 4, 64, 320, 2)
        s.step(_t([3, 1, 0, 17, 40], cuda), 61)
        return s

    eager, graphed = fresh(), fresh()
    new = torch.ones(5, dtype=torch.int32, device=cuda)
    inputs = torch.zeros((5, (8 + 4) * 128), dtype=dtype, device=cuda)
    side = torch.cuda.Stream()
    keep = [t.clone() for t in (graphed.table, graphed.lens, graphed.count, graphed.k, graphed.v)]
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graphed.step(new, 5, inputs)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = graphed.step(new, 5, inputs)[4]
    for t, was in zip((graphed.table, graphed.lens, graphed.count, graphed.k, graphed.v), keep):
        t.copy_(was)
    g = torch.Generator(cuda).manual_seed(9)
    for _ in range(12):
        x = torch.randn(inputs.shape, generator=g, device=cuda).to(dtype)
        want = eager.step(new, 5, x)[4]
        inputs.copy_(x)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(graphed.lens, eager.lens) and torch.equal(graphed.table, eager.table)


@pytest.mark.parametrize("n", [300, 6000])
def test_lengths_that_the_launch_before_writes(cuda, n):
    """The length and the page of the new token come from the kernel right before the attention."""
    q, k, v, table, lens = _case(cuda, torch.bfloat16, [n, 40, 7], 2, 4, 128, 16, spare=9, width=2)
    k.nan_to_num_(0.5), v.nan_to_num_(0.25)
    free = _t(sorted(set(range(k.shape[0])) - set(table.flatten().tolist())), cuda)
    count = _t([free.numel()], cuda)
    one = torch.ones(3, dtype=torch.int32, device=cuda)
    for _ in range(30):
        s = ops.PagedAdvance(table, lens, one, free, count, 16, 3, inplace=True)
        got = ops.PagedDecodeAttention(q, k, v, table, s.lens, 0.1)
        want, bound = paged_plain.attention(q, k, v, table, lens, 0.1)
        assert bool(((got.double() - want).abs() <= bound).all())


def test_two_streams_at_once(cuda):
    """Calls of two streams side by side, and again: each gets what it gets alone."""
    cases = [_case(cuda, torch.bfloat16, [n, 5, n // 3], 2, 4, 128, 16, seed=n) for n in (4000, 9000)]
    alone = [ops.PagedDecodeAttention(*c, 0.1) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(20):
        for i, (s, c) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(s):
                got[i].append(ops.PagedDecodeAttention(*c, 0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(x, a) for a, xs in zip(alone, got) for x in xs)


def test_two_graphs_at_once(cuda):
    """Two captured attentions replayed on two streams: neither uses the other's memory."""
    cases = [_case(cuda, torch.bfloat16, [n, 50], 1, 4, 128, 16, seed=n) for n in (20000, 15000)]
    alone = [ops.PagedDecodeAttention(*c, 0.1) for c in cases]
    graphs, outs = [], []
    for c in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.PagedDecodeAttention(*c, 0.1))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, a) for o, a in zip(outs, alone))
