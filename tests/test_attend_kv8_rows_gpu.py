"""Attention of many rows over the 8-bit cache (the form on tcgen05): shapes of its tiles, shares and sequences."""
import math

import pytest
import torch

from oxinfer_b200.kv8 import Kv8Seqs

from test_attend_kv8_gpu import DEV, Setting, i32, slopes_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv,counts", [(4, 4, [64]), (4, 4, [128]), (4, 4, [129]), (4, 4, [255, 256, 257]), (12, 4, [85]), (20, 4, [13]), (8, 1, [33, 100]), (2, 1, [64, 600])])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_rows_of_every_tile(backend, nh, nkv, counts, hd, dtype):
    """Tiles that are full, that have a row more or less, and heads that do not divide them; from an empty cache and behind keys."""
    Setting(backend, counts, counts, nh, nkv, hd, dtype, seed=sum(counts)).check()
    Setting(backend, [c + 129 for c in counts], counts, nh, nkv, hd, dtype, seed=sum(counts) + 1, spread=2.0).check()


@pytest.mark.parametrize("length,count", [(1000, 70), (4100, 64), (3000, 300), (9000, 128), (20001, 65)])
def test_shares_of_long_contexts(backend, length, count):
    for nh, nkv in ((1, 1), (8, 4)):
        s = Setting(backend, [length], [count], nh, nkv, 128, "bf16", seed=length, spread=2.0)
        s.check()
        s.check(window=300)  # (shares without keys in sight)
        s.check(window=37, prefix=[500])


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv,count", [(8, 8, 64), (16, 8, 33), (32, 8, 16), (40, 8, 13), (8, 8, 127), (32, 8, 63)])
def test_less_than_a_tile_of_several_sequences(backend, nh, nkv, count, hd):
    counts = [count, 1, 0, count - 3, count, 2]
    Setting(backend, [c + 40 * i + 1 for i, c in enumerate(counts)], counts, nh, nkv, hd, "bf16", seed=count, spread=2.0).check(cap=25.0)
    Setting(backend, [c + 40 * i + 1 for i, c in enumerate(counts)], counts, nh, nkv, hd, "f16", seed=count + 1).check()


def test_many_ragged_sequences(backend):
    """More than a warp looks through at once, some without rows, some with one."""
    counts = [(7 * i * i) % 90 for i in range(75)]
    lengths = [c + (13 * i) % 200 for i, c in enumerate(counts)]
    lengths = [max(1, n) for n in lengths]
    Setting(backend, lengths, counts, 4, 2, 64, "f16", seed=3).check()
    Setting(backend, lengths, counts, 4, 2, 64, "f16", seed=4, spread=3.0).check(cap=20.0, slopes=slopes_of(4), window=64, prefix=[(5 * i) % 100 for i in range(75)])


@pytest.mark.parametrize("cap,spread", [(50.0, 2.0), (50.0, 30.0), (5.0, 3.0), (0.25, 3.0), (30.0, 1e-3)])
def test_caps_over_every_range(backend, cap, spread):
    Setting(backend, [300, 150], [100, 150], 4, 2, 128, "bf16", seed=8, spread=spread).check(cap=cap)


def test_scores_that_grow_along_the_keys(backend):
    """The largest score of every row moves on from tile to tile, by less and by more than the sums wait for; and the other way round."""
    for slope in (0.05, 0.5, -0.05, -0.5):
        s = Setting(backend, [900], [300], 2, 1, 64, "f16", seed=9)
        s.check(slopes=torch.tensor([slope, slope / 3], device=DEV))


def test_scales_of_values_that_differ(backend):
    """Blocks whose values are 2^20 apart; rows that see the small ones only."""
    nkv, hd, n = 1, 64, 256
    s = Setting(backend, [n], [n], 2, nkv, hd, "bf16", seed=10)
    g = torch.Generator(device=DEV)
    g.manual_seed(1)
    size = torch.tensor([2.0 ** (20 * (i // 32 % 3 == 2) - 10 * (i // 32 % 3 == 1) - 15) for i in range(n)], device=DEV)
    v = torch.randn((n, nkv, hd), device=DEV, generator=g) * size[:, None, None]
    every = Kv8Seqs(start=i32([0]), max_rows=n, max_blocks=s.max_blocks, table=s.table)
    k = s.k.clone()
    assert s.cache.append(every, k, v) and s.cache.read(every, s.k, s.v)
    y, _ = s.want()
    out = torch.empty_like(s.q)
    assert s.cache.attend(s.seqs, s.q, out, scale=s.scale)
    # against the largest value in the row's own sight: 2^-11 of a probability, queries in f16 as they are (bf16 here: exact), half a step of the result
    j = torch.arange(n, device=DEV)
    seen = torch.cummax(s.v[:, 0].abs().amax(-1), 0).values.double()
    tol = (seen * (2.0 ** -11 + 2.0 ** -13))[:, None, None] + torch.finfo(torch.bfloat16).eps / 2 * y.abs()
    # (scores: 2^-18.5 of their magnitudes, below 2^-13 of a probability)
    assert ((out.double() - y).abs() <= tol).all(), ((out.double() - y).abs() / tol).max()
    assert (y[:32].abs().amax() < 2.0 ** -11) and torch.isfinite(out).all() and j.numel() == n


@pytest.mark.parametrize("shift", [0, 1, 4])
def test_strides_and_results_in_place(backend, shift):
    s = Setting(backend, [100, 177], [70, 150], 4, 2, 64, "f16", seed=12)
    want = s.check()
    width, rows = 4 * 64 + 8 + shift, s.n_rows
    room = torch.full((rows * width + shift,), 5.0, dtype=s.dtype, device=DEV)
    view = room.as_strided((rows, 4, 64), (width, 64, 1), shift)
    view.copy_(s.q)
    seqs = Kv8Seqs(start=s.seqs.start, rows=s.seqs.rows, n_rows=rows, max_rows=40, max_blocks=s.max_blocks, table=s.table)  # (a hint below the longest)
    assert s.cache.attend(seqs, view, view, scale=s.scale)
    assert torch.equal(view, want)
    left = torch.ones_like(room, dtype=torch.bool)
    left.as_strided((rows, 4, 64), (width, 64, 1), shift).fill_(False)
    assert (room[left] == 5.0).all()


def test_what_is_not_finite(backend):
    for kind in (0, 1):
        s = Setting(backend, [400, 90], [300, 64], 4, 2, 128, "bf16", seed=6, poison=[(0, 250, 1, kind), (1, 5, 0, kind)])
        out = s.check()
        assert torch.isnan(out[150:300, 2:]).all() and not torch.isnan(out[:150]).any() and not torch.isnan(out[150:300, :2]).any() and torch.isnan(out[300:, :2]).all()
        assert not torch.isnan(s.check(window=20)[171:300]).any()
    s = Setting(backend, [200], [100], 2, 1, 64, "f16", seed=7)
    clean = s.check()
    s.q[37, 1, 5], s.q[99, 0, 63] = math.inf, math.nan
    out = torch.empty_like(s.q)
    assert s.cache.attend(s.seqs, s.q, out, scale=s.scale)
    hit = torch.zeros((100, 2), dtype=torch.bool, device=DEV)
    hit[37, 1] = hit[99, 0] = True
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


def test_negative_and_zero_scales(backend):
    for scale in (-0.2, 0.0):
        s = Setting(backend, [300], [130], 2, 1, 64, "bf16", seed=15)
        s.scale = scale
        s.check()
        s.check(cap=4.0)


def test_captured(backend):
    s = Setting(backend, [500], [200], 4, 2, 64, "bf16", seed=16)
    want = s.check(cap=10.0)
    side, out = torch.cuda.Stream(), torch.empty_like(s.q)
    torch.cuda.synchronize()
    backend.set_stream(side.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            assert s.cache.attend(s.seqs, s.q, out, scale=s.scale, cap=10.0)
        for _ in range(3):
            out.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
    finally:
        backend.set_stream(0)
