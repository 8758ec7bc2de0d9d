"""Paged serving without a GPU: frequencies against their definitions, refusals of the operators and of the C entries, the oracle of the page
accounting against an independent account."""
import ctypes as C
import math
import random

import pytest
import torch

from light_b200 import _lib, ops
import paged_plain


def test_frequencies_plain_linear_and_ntk():
    f, m = ops.RoPEFrequencies(8, 10000.0, device="cpu")
    assert f.dtype == torch.float64 and m == 1.0
    for i, got in enumerate(f.tolist()):
        assert got == pytest.approx(math.exp(-2 * i / 8 * math.log(10000.0)), rel=1e-14)
    g, _ = ops.RoPEFrequencies(8, 10000.0, "linear", 4.0, device="cpu")
    assert torch.allclose(g * 4, f, rtol=1e-15)
    n, _ = ops.RoPEFrequencies(8, 10000.0, "ntk", 4.0, device="cpu")
    assert n[0] == f[0] and n[-1].item() == pytest.approx(f[-1].item() / 4, rel=1e-12)  # what the base is chosen for


def test_frequencies_llama3_and_yarn_keep_fast_pairs_and_stretch_slow_ones():
    base, original, factor = 500000.0, 8192, 8.0
    f, _ = ops.RoPEFrequencies(128, base, device="cpu")
    turns = original * f / (2 * math.pi)
    g, m = ops.RoPEFrequencies(128, base, "llama3", factor, original=original, device="cpu")
    assert m == 1.0
    for t, a, b in zip(turns.tolist(), f.tolist(), g.tolist()):
        wave = 2 * math.pi / a
        if wave < original / 4:
            want = a
        elif wave > original / 1:
            want = a / factor
        else:
            smooth = (original / wave - 1) / (4 - 1)
            want = (1 - smooth) * a / factor + smooth * a
        assert b == pytest.approx(want, rel=1e-13)
    y, m = ops.RoPEFrequencies(128, 10000.0, "yarn", 16.0, original=4096, device="cpu")
    f, _ = ops.RoPEFrequencies(128, 10000.0, device="cpu")
    turns = (4096 * f / (2 * math.pi)).tolist()
    assert m == pytest.approx(0.1 * math.log(16) + 1)
    ratio = (y / f).tolist()
    assert all(r == pytest.approx(1.0, rel=1e-12) for r, t in zip(ratio, turns) if t > 33 * 1.2)
    assert all(r == pytest.approx(1 / 16, rel=1e-12) for r, t in zip(ratio, turns) if t < 1 / 1.2)
    assert all(b <= a * (1 + 1e-12) for a, b in zip(ratio, ratio[1:]))


@pytest.mark.parametrize("args,kw", [((7, 1e4), {}), ((0, 1e4), {}), ((8, 0.0), {}), ((8, 1e4, "linear", 0.0), {}), ((8, 1e4, "yarn", 2.0), {}), ((8, 1e4, "llama3", 2.0), {}),
                                     ((2, 1e4, "ntk", 2.0), {}), ((8, 1e4, "dynamic", 2.0), {}), ((8, 1.0, "yarn", 2.0), {"original": 4096}),
                                     ((8, 1e4, "llama3", 2.0), {"original": 4096, "low": 4.0, "high": 4.0})])
def test_frequencies_refusals(args, kw):
    with pytest.raises(ValueError, match="RoPEFrequencies"):
        ops.RoPEFrequencies(*args, device="cpu", **kw)


def test_operators_refuse_cpu_tensors():
    t, i = torch.zeros(2, 4, 8), torch.zeros(2, dtype=torch.int32)
    cache, table = torch.zeros(3, 4, 16, 8), torch.zeros((2, 3), dtype=torch.int32)
    for call in (lambda: ops.PagedDecodeAttention(t, cache, cache, table, i, 1.0),
                 lambda: ops.QKNormRoPE(t, t, torch.zeros(2, dtype=torch.int64), torch.ones(4, dtype=torch.float64)),
                 lambda: ops.PagedAdvance(table, i, i, i, i[:1], 16, 2),
                 lambda: ops.PagedRelease(table, i, i > 0, i, i[:1], 16)):
        with pytest.raises(ValueError, match="CUDA kernels only"):
            call()


def _attn_args(**kw):
    a = dict(q=256, k=256, v=256, block_table=256, lens=256, out=256, q_stride=(256, 64), k_stride=(8192, 1024, 64), v_stride=(8192, 1024, 64), table_stride=4, pages=5, dtype=0, B=2,
             NH=4, KH=2, D=64, page_size=16, W=4, window=0, scale=1.0, softcap=0.0)
    a.update(kw)
    a = {n: (C.c_int64 * len(v))(*v) if isinstance(v, tuple) else v for n, v in a.items()}
    return _lib.PagedAttnArgs(**a)


@pytest.mark.parametrize("kw,code", [(dict(dtype=7), -1), (dict(NH=5), -2), (dict(D=0), -2), (dict(D=257), -2), (dict(W=0), -2), (dict(pages=0), -2), (dict(page_size=0), -2),
                                     (dict(window=-1), -2), (dict(table_stride=3), -2), (dict(softcap=-1.0), -2), (dict(softcap=float("nan")), -2),
                                     (dict(W=1 << 27, page_size=16, table_stride=1 << 27), -6), (dict(lens=0), -3), (dict(q=0), -3), (dict(B=-1), -2)])
def test_attention_entry_refuses(kw, code):
    assert _lib.lib().light_b200_paged_decode_attn(C.byref(_attn_args(**kw)), 0, None) == code
    assert "paged_decode_attn" in _lib.last_error()
    assert _lib.lib().light_b200_paged_attn_scratch_bytes(C.byref(_attn_args(**kw)), 0) == 0
    assert _lib.lib().light_b200_paged_decode_attn(None, 0, None) == -3


@pytest.mark.parametrize("softcap", [float("inf"), 3e38, 1.1e20, 9e-21, 1e-38])
def test_attention_entry_refuses_caps_that_overflow(softcap):
    """scale / cap and cap log2 e are f32: an infinite one would turn scores into NaN."""
    assert _lib.lib().light_b200_paged_decode_attn(C.byref(_attn_args(softcap=softcap)), 0, None) == -2


def _rope_args(**kw):
    a = dict(q=256, k=256, q_out=256, k_out=256, positions=256, inv_freq=256, q_stride=(256, 64), k_stride=(128, 64), T=3, dtype=1, NH=4, KH=2, D=64, rotary=64, page_size=1, eps=1e-6,
             factor=1.0)
    a.update(kw)
    a = {n: (C.c_int64 * len(v))(*v) if isinstance(v, tuple) else v for n, v in a.items()}
    return _lib.QKNormRopeArgs(**a)


@pytest.mark.parametrize("kw,code", [(dict(dtype=5), -1), (dict(D=257), -2), (dict(rotary=63), -2), (dict(rotary=66), -2), (dict(rotary=-2), -2), (dict(NH=0), -2), (dict(KH=0), -2),
                                     (dict(T=-1), -2), (dict(T=1 << 31), -6), (dict(eps=-1.0), -2), (dict(eps=float("nan")), -2), (dict(slots=256), -2),
                                     (dict(slots=256, pages=4, page_size=16), -3), (dict(positions=0), -3), (dict(inv_freq=0), -3), (dict(k_out=0), -3)])
def test_rotation_entry_refuses(kw, code):
    assert _lib.lib().light_b200_qk_norm_rope(C.byref(_rope_args(**kw)), 0, None) == code
    assert "qk_norm_rope" in _lib.last_error()
    assert _lib.lib().light_b200_qk_norm_rope(None, 0, None) == -3


def _pages(**kw):
    a = {n: 256 for n in ("block_table", "lens", "new_lens", "done", "free_pages", "free_count", "lens_out", "granted", "starts", "free_count_out", "positions", "slots")}
    a.update(table_stride=4, tokens=8, B=2, W=4, page_size=16, capacity=9)
    a.update(kw)
    return _lib.PagedPages(**a)


@pytest.mark.parametrize("kw,code", [(dict(B=0), -2), (dict(W=0), -2), (dict(page_size=0), -2), (dict(capacity=0), -2), (dict(tokens=-1), -2), (dict(table_stride=3), -2),
                                     (dict(B=8193), -6), (dict(W=1 << 28, table_stride=1 << 28), -6), (dict(tokens=1 << 31), -6), (dict(lens=0), -3), (dict(free_count_out=0), -3)])
def test_page_entries_refuse(kw, code):
    for f, own in (("light_b200_paged_advance", dict(slots=0)), ("light_b200_paged_release", dict(done=0))):
        assert getattr(_lib.lib(), f)(C.byref(_pages(**kw)), 0, None) == code
        assert getattr(_lib.lib(), f)(C.byref(_pages(**own)), 0, None) == -3
        assert getattr(_lib.lib(), f)(None, 0, None) == -3


def test_argument_blocks_match_the_header(tmp_path):
    import shutil
    import subprocess

    from helpers import ROOT

    if shutil.which("gcc") is None:
        pytest.skip("no C compiler")
    src = tmp_path / "s.c"
    names = {"lb200_paged_pages": _lib.PagedPages, "lb200_qk_norm_rope_args": _lib.QKNormRopeArgs, "lb200_paged_attn_args": _lib.PagedAttnArgs}
    body = "".join(f'printf("%zu ", sizeof({n}));' + "".join(f'printf("%zu ", offsetof({n}, {f[0]}));' for f in c._fields_) for n, c in names.items())
    src.write_text(f'#include "{ROOT}/include/light_b200.h"\n#include <stdio.h>\nint main(void) {{ {body} return 0; }}\n')
    subprocess.run(["gcc", str(src), "-o", str(tmp_path / "s")], check=True)
    got = list(map(int, subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()))
    want = [x for c in names.values() for x in [C.sizeof(c)] + [getattr(c, f[0]).offset for f in c._fields_]]
    assert got == want


def test_oracle_of_the_pages_never_hands_one_out_twice():
    """A pool under random arrivals and departures: every page is free or belongs to one request, and the slots of a request are its tokens in order."""
    rng = random.Random(3)
    page, width, pool, B = 4, 6, 20, 5
    free, count = list(range(pool)), pool
    table, lens = [[-1] * width for _ in range(B)], [0] * B
    rows = [[] for _ in range(B)]
    for _ in range(200):
        new = [rng.choice([0, 1, 1, 1, 7]) for _ in range(B)]
        pos, slot, starts, lens, given, count = paged_plain.advance(table, lens, new, free, count, page, sum(new) + 2)
        for b in range(B):
            for i in range(given[b]):
                assert pos[starts[b] + i] == len(rows[b])
                rows[b].append(slot[starts[b] + i])
        done = [rng.random() < 0.1 for _ in range(B)]
        for b in range(B):
            assert len(rows[b]) == lens[b] and len(set(rows[b])) == lens[b]
            assert rows[b] == [table[b][j // page] * page + j % page for j in range(lens[b])]
        held = [p for b in range(B) for p in table[b][:-(-lens[b] // page)]]
        assert sorted(held + free[:count]) == list(range(pool))
        lens, count = paged_plain.release(table, lens, done, free, count, page)
        rows = [[] if d else r for r, d in zip(rows, done)]
