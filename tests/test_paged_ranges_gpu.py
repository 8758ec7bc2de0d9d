"""The paged operators where their ranges end: weights far below the largest, fewer query heads than key heads, angles next to a zero of the cosine,
pools that hold what no pool should, the largest sizes."""
import math

import paged_plain
import pytest
import torch

from light_b200 import _lib, ops

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def _dense(scores, v, KH, G, D, dtype, dev, page=16, width=0):
    """One sequence per row of `scores` (B, n): key j's first element is its score, query heads look at nothing else, so scores are exact; v (B, n)
    or (B, n, D) are the values of all heads."""
    B, n = scores.shape
    held = -(-n // page)
    k_cache, v_cache = (torch.zeros((B * held, KH, page, D), dtype=dtype, device=dev) for _ in range(2))
    table = torch.full((B, held + width), -1, dtype=torch.int32, device=dev)
    table[:, :held] = torch.arange(B * held, device=dev).view(B, held)
    pad = torch.zeros((B, held * page), dtype=dtype, device=dev)
    pad[:, :n] = scores.to(dtype)
    k_cache[..., 0] = pad.view(B * held, 1, page)
    rows = torch.zeros((B, held * page, D), dtype=dtype, device=dev)
    rows[:, :n] = v.to(dtype)[..., None] if v.dim() == 2 else v.to(dtype)
    v_cache[:] = rows.view(B * held, 1, page, D)
    q = torch.zeros((B, KH * G, D), dtype=dtype, device=dev)
    q[..., 0] = 1
    return q, k_cache, v_cache, table, torch.full((B,), n, dtype=torch.int32, device=dev)


def _close(case, rounded_p=False, **kw):
    """Within the arithmetic's bound, for weights that lose nothing to the cache's type, or (rounded_p) no more than one rounding each."""
    got = ops.PagedDecodeAttention(*case, 1.0, **kw)
    want, bound = paged_plain.attention(*case, 1.0, rounded_p=rounded_p, **kw)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), (off / bound.clamp(min=1e-300)).max().item()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("at", ["first", "last", "within"])
@pytest.mark.parametrize("n,B,D", [(300, 1, 128), (8192, 3, 128), (8192, 40, 64), (131072, 1, 128), (1000, 2, 256), (500, 3, 37), (20000, 1, 80)])
def test_light_keys_under_a_heavy_one(cuda, dtype, at, n, B, D):
    """A key with nearly all of the weight and a value of zero: the answer is the sum of what the others weigh, however little each does."""
    for binades in (10.0, 14.5, 20.0, 21.0, 22.0, 24.5, 26.0, 30.0, 40.0, 70.0):
        s = torch.zeros((B, n), dtype=torch.float64, device=cuda)
        s[:, 1::2] = -1.0
        v = torch.full((B, n), 1.0, dtype=torch.float64, device=cuda)
        v[:, ::3] = 3.0
        if dtype != torch.bfloat16:
            v *= 2.0 ** 12  # (so that the answer is no subnormal half)
        j = {"first": 0, "last": n - 1, "within": min(n // 2 + 3, n - 1)}[at]
        s[:, j], v[:, j] = binades * math.log(2), 0.0
        _close(_dense(s, v, 1, 3, D, dtype, cuda), rounded_p=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [1, 9])
def test_weights_of_every_size_side_by_side(cuda, dtype, G):
    """Neighbouring keys 0 to 60 binades apart, each size with a value that makes it count; windows and caps among them."""
    g = torch.Generator(cuda).manual_seed(G)
    s = -torch.randint(0, 61, (6, 700), generator=g, device=cuda).double() * math.log(2)
    v = torch.randn((6, 700, 64), generator=g, device=cuda).double() * torch.exp(-s).clamp(max=2.0 ** 13)[..., None]
    for kw in ({}, {"window": 100}, {"softcap": 50.0}):
        _close(_dense(s, v, 2, G, 64, dtype, cuda), rounded_p=True, **kw)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G,width", [(4, 0), (12, 0), (4, 3000)])
@pytest.mark.parametrize("far", [0.0, 5.0, 17.0, 30.0, 40.0])
def test_infinite_values_reach_their_heads_with_their_sign(cuda, dtype, G, width, far):
    """A value of infinity under a weight that is not 0 is the result; opposite ones, or one under a weight of 0 (its score -inf), are NaN."""
    s = torch.zeros((5, 200), dtype=torch.float64, device=cuda)
    s[:, 7] = far
    v = torch.ones((5, 200, 64), dtype=torch.float64, device=cuda)
    v[0, 3, 0] = v[1, 7, 1] = v[3, 3, 2] = v[4, 3, 2] = math.inf
    v[1, 150, 2] = v[3, 150, 2] = -math.inf
    s[4, 3] = -math.inf
    got = ops.PagedDecodeAttention(*_dense(s, v, 2, G, 64, dtype, cuda, width=width), 1.0).double()
    odd = torch.zeros_like(got)
    odd[0, :, 0] = odd[1, :, 1] = math.inf
    odd[1, :, 2] = -math.inf
    odd[3, :, 2] = odd[4, :, 2] = math.nan
    assert torch.equal(got.isnan(), odd.isnan())
    assert torch.equal(torch.where(got.isinf(), got, 0), torch.where(odd.isinf(), odd, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("G", [1, 12])
@pytest.mark.parametrize("B,n", [(1, 2), (9, 64), (40, 1500)])
def test_weights_are_as_exact_as_the_scores(cuda, dtype, G, B, n):
    """Pairs of keys whose weighted values cancel: what a weight's rounding to the cache's type would leave over is far above the bound."""
    g = torch.Generator(cuda).manual_seed(n)
    s = (torch.rand((B, n), generator=g, device=cuda) * 3).to(dtype).double()
    v = torch.ones((B, n), dtype=torch.float64, device=cuda)
    v[:, 1::2] = -torch.exp(s[:, 0::2] - s[:, 1::2])
    _close(_dense(s, v, 2, G, 64, dtype, cuda))
    _close(_dense(s, v, 2, G, 64, dtype, cuda), softcap=20.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("down", [0.0, 9.0, 25.0])
def test_weights_under_a_heavy_one_are_as_exact(cuda, dtype, down):
    """The same under a key of value 0 that is `down` nats above the others; far below it halves have
    products of their own."""
    g = torch.Generator(cuda).manual_seed(5)
    s = (-down - torch.rand((5, 400), generator=g, device=cuda) * 3).to(dtype).double()
    v = torch.ones((5, 400), dtype=torch.float64, device=cuda)
    v[:, 1::2] = -torch.exp(s[:, 0::2] - s[:, 1::2])
    s[:, 0], v[:, :2] = 0.0, 0.0
    v *= 2.0 ** 11
    _close(_dense(s, v, 2, 4, 64, dtype, cuda))
    _close(_dense(s, v, 2, 12, 64, dtype, cuda, width=3000))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 500, 600, 1000, 1700, 2000])
@pytest.mark.parametrize("NH,KH,D", [(4, 8, 128), (1, 8, 128), (4, 5, 128), (2, 16, 128), (8, 16, 64), (1, 40, 64), (3, 20, 80), (1, 3, 256)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_of_fewer_query_heads_than_key_heads(cuda, dtype, T, NH, KH, D, interleaved):
    g = torch.Generator(cuda).manual_seed(T + NH)
    q, k, v = (torch.randn((T, n, D), generator=g, device=cuda).to(dtype) for n in (NH, KH, KH))
    w = (1 + 0.2 * torch.randn(D, generator=g, device=cuda)).to(dtype)
    freq, _ = ops.RoPEFrequencies(D, 10000.0)
    positions = torch.arange(T, device=cuda)
    pages = T // 16 + 1
    kc, vc = (torch.zeros((pages, KH, 16, D), dtype=dtype, device=cuda) for _ in range(2))
    slots = torch.randperm(pages * 16, generator=g, device=cuda)[:T].contiguous()
    got, _ = ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=w, interleaved=interleaved, v=v, k_cache=kc, v_cache=vc, slots=slots)
    again, dense = ops.QKNormRoPE(q, k, positions, freq, q_weight=w, k_weight=w, interleaved=interleaved)
    want, bound = paged_plain.rotated(q, w, 1e-6, positions, freq, interleaved, 1.0)
    assert bool(((got.double() - want).abs() <= bound).all()) and torch.equal(again, got)
    want, bound = paged_plain.rotated(k, w, 1e-6, positions, freq, interleaved, 1.0)
    assert bool(((dense.double() - want).abs() <= bound).all())
    assert torch.equal(kc[slots // 16, :, slots % 16], dense) and torch.equal(vc[slots // 16, :, slots % 16], v)


@pytest.mark.parametrize("D", [64, 7])
@pytest.mark.parametrize("interleaved", [False, True])
def test_rotation_keeps_sines_and_cosines_next_to_their_zeros(cuda, D, interleaved):
    """Angles within 1e-6 of whole quarter turns, near and far from the start: the sine or cosine that is nearly zero has its own precision."""
    R = D // 2 * 2
    positions = torch.tensor([1, 3, 1001, 100003], device=cuda)
    quarter = torch.arange(R // 2, dtype=torch.float64, device=cuda)
    freq = (quarter % 7) * (math.pi / 2) + (0.1 + quarter) * 1e-11
    q = torch.zeros((4, 3, D), device=cuda)
    first = slice(0, R, 2) if interleaved else slice(0, R // 2)
    q[:, :, first] = torch.tensor([1.0, -0.5, 3.0], device=cuda)[None, :, None]
    got, _ = ops.QKNormRoPE(q, q, positions, freq, interleaved=interleaved)
    t = positions.double()[:, None, None] * freq
    a = q[:, :, first].double()
    second = slice(1, R, 2) if interleaved else slice(R // 2, R)
    # The angle in 64 bits has four roundings of 2^-53 (here one, there three); sine and cosine of an f32 angle at most pi 2^-25 away are right to two
    # steps of 2^-23, as are the products and the sum that bring them there.
    for part, want in ((first, a * torch.cos(t)), (second, a * torch.sin(t))):
        bound = 4 * 2.0 ** -53 * t.abs() * a.abs() + 8 * 2.0 ** -23 * (want.abs() + 2.0 ** -23 * a.abs())
        off = (got[:, :, part].double() - want).abs()
        assert bool((off <= bound).all()), (off / bound.clamp(min=1e-300)).max().item()


def _i32(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def test_status_is_read_and_cleared(cuda):
    """Each bit is met, read, read again and cleared; the next fault behind it shows."""
    q, cache = torch.zeros((1, 2, 64), device=cuda), torch.zeros((2, 2, 8, 64), device=cuda)
    table, one, none = _i32([[0, 1]], cuda), _i32([1], cuda), _i32([0], cuda)
    pos, freq = torch.zeros(1, dtype=torch.int64, device=cuda), ops.RoPEFrequencies(64, 1e4)[0]
    met = {1: lambda: ops.PagedDecodeAttention(q, cache, cache, table, _i32([17], cuda), 1.0),
           2: lambda: ops.PagedDecodeAttention(q, cache, cache, _i32([[2, 0]], cuda), one, 1.0),
           4: lambda: ops.QKNormRoPE(q, q, pos, freq, v=q, k_cache=cache.clone(), v_cache=cache.clone(), slots=pos + 16),
           8: lambda: ops.PagedAdvance(table, none, one, one, none, 8, 1)}
    ops.paged_status(0, clear=True)
    for _ in range(2):
        for bit, call in met.items():
            call()
            assert ops.paged_status(0) == bit and ops.paged_status(0, clear=True) == bit and ops.paged_status(0) == 0
    for call in met.values():
        call()
    assert ops.paged_status(0, clear=True) == 15 and ops.paged_status(0, clear=True) == 0


def test_advance_of_nearly_two_to_the_31_pages(cuda):
    """8192 prompts of 262143 tokens, a page each: what counts pages must not wrap around."""
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("not enough memory")
    B, n = 8192, (1 << 18) - 1
    total = B * n
    table = torch.full((B, n + 1), -1, dtype=torch.int32, device=cuda)
    free = torch.arange(total + 5, dtype=torch.int32, device=cuda)
    new = torch.full((B,), n, dtype=torch.int32, device=cuda)
    s = ops.PagedAdvance(table, torch.zeros_like(new), new, free, _i32([total + 5], cuda), 1, total)
    assert s.free_count.tolist() == [5] and bool((s.granted == n).all()) and bool((s.lens == n).all()) and bool((table[:, n] == -1).all())
    at = torch.arange(n, device=cuda)
    for b in range(0, B, 256):
        rows = (torch.arange(b, b + 256, device=cuda) * n)[:, None] + at
        assert bool((s.positions[b * n:(b + 256) * n].view(256, n) == at).all())
        assert bool((s.slots[b * n:(b + 256) * n].view(256, n) == total + 4 - rows).all())
        assert bool((table[b:b + 256, :n] == total + 4 - rows).all())
    del s, table, free
    torch.cuda.empty_cache()


@pytest.mark.parametrize("B", [3, 3000])
@pytest.mark.parametrize("inplace", [False, True])
def test_pages_below_zero_are_reported(cuda, B, inplace):
    """A hole in a held page's place, on the stack, and on its way back to it: nothing of it goes by in silence."""
    def step(held, free, done):
        table = torch.full((B, 3), 7, dtype=torch.int32, device=cuda)
        table[B - 1, 0] = held
        lens, one = torch.zeros(B, dtype=torch.int32, device=cuda), torch.zeros(B, dtype=torch.int32, device=cuda)
        lens[B - 1], one[B - 1], one[0] = 3, 1, 1
        stack, count = _i32([1, free, 3], cuda), _i32([2], cuda)
        s = ops.PagedAdvance(table, lens, one, stack, count, 4, 2, inplace=inplace)
        given = (s.granted.tolist()[0], s.granted.tolist()[-1], s.slots.tolist(), ops.paged_status(0, clear=True))
        ops.PagedRelease(table, s.lens, torch.arange(B, device=cuda) == (B - 1 if done else B), stack, s.free_count, 4, inplace=inplace)
        return given, ops.paged_status(0, clear=True)
    ops.paged_status(0, clear=True)
    assert step(5, 2, True) == ((1, 1, [8, 23], 0), 0)
    assert step(-1, 2, False) == ((1, 1, [8, -1], 8), 0)
    assert step(-1, 2, True) == ((1, 1, [8, -1], 8), 8)
    assert step(5, -4, False) == ((1, 1, [-1, 23], 8), 0)


def test_attention_refuses_scales_that_overflow(cuda):
    q, cache = torch.zeros((1, 2, 64), device=cuda), torch.ones((2, 2, 8, 64), device=cuda)
    table, lens = _i32([[0, 1]], cuda), _i32([9], cuda)
    for scale, cap in ((1e19, 1e-20), (3e38, 0.0), (math.inf, 0.0), (math.nan, 5.0)):
        with pytest.raises(ValueError, match="scale"):
            ops.PagedDecodeAttention(q, cache, cache, table, lens, scale, softcap=cap)
    for scale, cap in ((1e18, 1e-20), (1e38, 0.0), (-1e38, 1e20), (1e-38, 1e20)):  # all scores 0: the mean of the values
        assert bool((ops.PagedDecodeAttention(q, cache, cache, table, lens, scale, softcap=cap) == 1).all())


@pytest.mark.parametrize("tokens", [1 << 31, 1 << 40, 1 << 60, 1 << 63])
def test_advance_refuses_more_tokens_than_it_counts_before_it_allocates(cuda, tokens):
    held = torch.cuda.memory_reserved()
    with pytest.raises(ValueError, match="PagedAdvance"):
        ops.PagedAdvance(_i32([[0, 1]], cuda), _i32([0], cuda), _i32([1], cuda), _i32([2], cuda), _i32([1], cuda), 16, tokens)
    assert torch.cuda.memory_reserved() - held < 1 << 30
