"""The 8-bit cache (b2_kv8_*): what rows stand for, bit for bit against the definition in 64 bits, whatever blocks they fall into."""
import numpy as np
import pytest
import torch

import oxinfer_b200 as ob
from oxinfer_b200.kv8 import BLOCK, Kv8Seqs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


class Model:
    """The definition: integers, a power of two a block, head and kind, rows that are not finite. Positions of one sequence."""

    def __init__(self, nkv, hd, blocks):
        self.q = np.zeros((blocks, 2, nkv, BLOCK, hd))
        self.scale = np.zeros((blocks, 2, nkv))
        self.bad = np.zeros((blocks, 2, nkv, BLOCK), bool)

    def append(self, start, k, v):
        for kind, x in enumerate((k, v)):
            for b in range(start // BLOCK, (start + len(x) - 1) // BLOCK + 1):
                lo, hi = max(start - b * BLOCK, 0), min(start + len(x) - b * BLOCK, BLOCK)
                new = x[b * BLOCK + lo - start:b * BLOCK + hi - start].astype(np.float64)  # [rows][nkv][hd]
                for h in range(x.shape[1]):
                    rows = new[:, h]
                    fine = np.isfinite(rows).all(1)
                    top = np.abs(rows[fine]).max() if fine.any() else 0.0
                    e = -100
                    while top > 127.0 * 2.0 ** e:
                        e += 1
                    scale = 2.0 ** e
                    most = 63 if e == 122 else 127  # (64 * 2^122 is no f32)
                    if lo:
                        scale = max(scale, self.scale[b, kind, h])
                        most = 63 if scale == 2.0 ** 122 else 127
                        self.q[b, kind, h, :lo] = np.clip(np.rint(self.q[b, kind, h, :lo] * (self.scale[b, kind, h] / scale)), -most, most)
                    self.scale[b, kind, h] = scale
                    self.q[b, kind, h, lo:hi] = np.where(fine[:, None], np.clip(np.rint(np.where(fine[:, None], rows, 0.0) / scale), -most, most), 0.0)
                    self.bad[b, kind, h, lo:hi] = ~fine

    def values(self, n):
        x = np.where(self.bad[..., None], np.nan, self.q * self.scale[..., None, None])
        x = x.transpose(1, 0, 3, 2, 4).reshape(2, -1, x.shape[2], x.shape[4])
        return x[0, :n], x[1, :n]


def read(cache, start, count, max_blocks, table=None):
    n = sum(count)
    k, v = (torch.full((n, cache.nkv, cache.hd), -7.0, device=DEV) for _ in range(2))
    rows = i32(np.concatenate([[0], np.cumsum(count)]))
    assert cache.read(Kv8Seqs(start=i32(start), rows=rows, n_rows=n, max_rows=max(count), max_blocks=max_blocks, table=table), k, v)
    return k.cpu().numpy().astype(np.float64), v.cpu().numpy().astype(np.float64)


def rows_of(rng, n, nkv, hd, dtype):
    x = torch.from_numpy((rng.standard_normal((n, nkv, hd)) * np.exp(rng.normal(0, 1.5, (n, 1, 1)))).astype(np.float32)).to(dtype)
    return x


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=["f32", "bf16", "f16"])
def test_appends_of_every_shape(backend, hd, dtype):
    """One sequence: rows one by one, in chunks that end inside blocks, over several blocks, back to an earlier position, and from a block's beginning anew."""
    nkv, blocks = 3, 6
    rng = np.random.default_rng(11 + hd)
    cache, model = backend.kv8(nkv, hd, blocks), Model(nkv, hd, blocks)
    end = 0
    for start, n in [(0, 1), (1, 1), (2, 3), (5, 7), (12, 20), (32, 31), (63, 1), (64, 33), (97, 40), (130, 5), (96, 2), (98, 64), (64, 1), (65, 126), (191, 1), (0, 192)]:
        k, v = (rows_of(rng, n, nkv, hd, dtype) for _ in range(2))
        assert cache.append(Kv8Seqs(start=i32([start]), max_rows=n, max_blocks=blocks), k.to(DEV), v.to(DEV))
        model.append(start, k.float().numpy(), v.float().numpy())
        end = start + n
        got, want = read(cache, [0], [end], blocks), model.values(end)
        for g, w in zip(got, want):
            assert np.array_equal(g, w), (start, n)
    backend.check_status()


def test_ragged_sequences_share_a_pool_through_their_tables(backend):
    nkv, hd, n_seqs, max_blocks = 2, 128, 5, 9
    rng = np.random.default_rng(5)
    table = rng.permutation(n_seqs * max_blocks + 3)[:n_seqs * max_blocks].reshape(n_seqs, max_blocks)
    cache, models = backend.kv8(nkv, hd, n_seqs * max_blocks + 3), [Model(nkv, hd, max_blocks) for _ in range(n_seqs)]
    held = [0] * n_seqs
    for counts in ([3, 0, 64, 33, 1], [1, 1, 1, 1, 1], [0, 200, 31, 0, 2], [7, 8, 9, 63, 65]):
        first = np.concatenate([[0], np.cumsum(counts)])
        k, v = (rows_of(rng, first[-1], nkv, hd, torch.float32) for _ in range(2))
        # (a hint below the longest sequence costs time and nothing else)
        seqs = Kv8Seqs(start=i32(held), rows=i32(first), n_rows=int(first[-1]), max_rows=max(1, max(counts) // 3), max_blocks=max_blocks, table=i32(table))
        assert cache.append(seqs, k.to(DEV), v.to(DEV))
        for s in range(n_seqs):
            if counts[s]:
                models[s].append(held[s], k[first[s]:first[s + 1]].numpy(), v[first[s]:first[s + 1]].numpy())
            held[s] += counts[s]
    for s in range(n_seqs):
        # from the middle of a block, too
        for start in (0, held[s] // 2):
            got = read(cache, [start], [held[s] - start], max_blocks, i32(table[s:s + 1]))
            for g, w in zip(got, models[s].values(held[s])):
                assert np.array_equal(g, w[start:]), (s, start)
    backend.check_status()


@pytest.mark.parametrize("hd,n_seqs,most", [(64, 5, 4), (128, 5, 6), (128, 130, 3), (64, 130, 8), (128, 130, 9)])
def test_a_few_rows_of_every_sequence(backend, hd, n_seqs, most):
    """Steps of up to `most` rows, some without one and some with one that is not finite: written, and read back alone, across the ends of blocks."""
    nkv, max_blocks = 8, 3
    rng = np.random.default_rng(n_seqs + most)
    cache, models = backend.kv8(nkv, hd, n_seqs * max_blocks), [Model(nkv, hd, max_blocks) for _ in range(n_seqs)]
    held = [int(v) for v in rng.integers(0, 40, n_seqs)]
    first = np.concatenate([[0], np.cumsum(held)])
    k, v = (rows_of(rng, first[-1], nkv, hd, torch.float32) for _ in range(2))
    assert cache.append(Kv8Seqs(start=i32([0] * n_seqs), rows=i32(first), n_rows=int(first[-1]), max_rows=40, max_blocks=max_blocks), k.to(DEV), v.to(DEV))
    for s in range(n_seqs):
        if held[s]:
            models[s].append(0, k[first[s]:first[s + 1]].numpy(), v[first[s]:first[s + 1]].numpy())
    for step in range(3):
        counts = [int(c) for c in rng.integers(0, most + 1, n_seqs)]
        counts[step] = most
        first = np.concatenate([[0], np.cumsum(counts)])
        k, v = (rows_of(rng, first[-1], nkv, hd, torch.float32) for _ in range(2))
        k[first[step], 2, 5], v[first[step], 7, 63] = np.inf, np.nan
        seqs = Kv8Seqs(start=i32(held), rows=i32(first), n_rows=int(first[-1]), max_rows=most, max_blocks=max_blocks)
        assert cache.append(seqs, k.to(DEV), v.to(DEV))
        got = [torch.full((int(first[-1]), nkv, hd), -7.0, device=DEV) for _ in range(2)]
        assert cache.read(seqs, *got)
        got = [x.cpu().numpy().astype(np.float64) for x in got]
        for s in range(n_seqs):
            if counts[s]:
                models[s].append(held[s], k[first[s]:first[s + 1]].numpy(), v[first[s]:first[s + 1]].numpy())
                for g, w in zip(got, models[s].values(held[s] + counts[s])):
                    assert np.array_equal(g[first[s]:first[s + 1]], w[held[s]:], equal_nan=True), (step, s)
            held[s] += counts[s]
    got = read(cache, [0] * n_seqs, held, max_blocks)
    first = np.concatenate([[0], np.cumsum(held)])
    for s in range(n_seqs):
        for g, w in zip(got, models[s].values(held[s])):
            assert np.array_equal(g[first[s]:first[s + 1]], w, equal_nan=True), s
    backend.check_status()


def test_magnitudes_from_zero_to_the_largest(backend):
    nkv, hd = 1, 64
    tops = [0.0, 1e-45, 1e-38, 127 * 2.0 ** -100, 126.9999 * 2.0 ** -100, 127.0, np.nextafter(np.float32(127.0), np.float32(200)), 128.0, 254.0, 1e30, np.finfo(np.float32).max]
    for i, top in enumerate(tops):
        cache, model = backend.kv8(nkv, hd, 1), Model(nkv, hd, 1)
        x = np.linspace(-1, 1, 3 * hd, dtype=np.float32).reshape(3, 1, hd) * np.float32(top)
        for start, rows in ((0, x[:2]), (2, x[2:] * np.float32(0.001)), (3, np.ones((1, 1, hd), np.float32))):
            assert cache.append(Kv8Seqs(start=i32([start]), max_rows=len(rows), max_blocks=1), *(torch.from_numpy(rows).to(DEV),) * 2)
            model.append(start, rows, rows)
            got = read(cache, [0], [start + len(rows)], 1)
            for g, w in zip(got, model.values(start + len(rows))):
                assert np.array_equal(g, w), (i, start)


def test_rows_that_are_not_finite_count_as_nan_and_leave_the_others_alone(backend):
    nkv, hd = 2, 128
    rng = np.random.default_rng(8)
    cache, model = backend.kv8(nkv, hd, 3), Model(nkv, hd, 3)
    k, v = (rows_of(rng, 70, nkv, hd, torch.float32) for _ in range(2))
    k[5, 0, 17], k[33, 1, 127], v[5, 1, 0], v[69, 0, 64] = np.inf, np.nan, -np.inf, np.nan
    assert cache.append(Kv8Seqs(start=i32([0]), max_rows=70, max_blocks=3), k.to(DEV), v.to(DEV))
    model.append(0, k.numpy(), v.numpy())
    for g, w in zip(read(cache, [0], [70], 3), model.values(70)):
        assert np.isnan(w).any() and np.array_equal(g, w, equal_nan=True)
    # a step that goes back behind them writes over them, one that goes on keeps them
    k2, v2 = (rows_of(rng, 2, nkv, hd, torch.float32) for _ in range(2))
    for start in (70, 33, 5):
        assert cache.append(Kv8Seqs(start=i32([start]), max_rows=2, max_blocks=3), k2.to(DEV), v2.to(DEV))
        model.append(start, k2.numpy(), v2.numpy())
        for g, w in zip(read(cache, [0], [start + 2], 3), model.values(start + 2)):
            assert np.array_equal(g, w, equal_nan=True), start


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shift,order", [(0, "rows"), (1, "rows"), (0, "heads"), (3, "heads")])
def test_strides_and_alignments(backend, dtype, shift, order):
    """Rows inside wider ones (a q / k / v vector), a head's rows side by side, and addresses aligned to an element only."""
    nkv, hd, n = 2, 64, 37
    rng = np.random.default_rng(21)
    k, v = (rows_of(rng, n, nkv, hd, dtype) for _ in range(2))
    put = []
    for x in (k, v):
        if order == "rows":
            room = torch.zeros(n * (nkv * hd + 8 + shift) + shift, dtype=dtype, device=DEV)
            view = room[shift:].as_strided((n, nkv, hd), (nkv * hd + 8 + shift, hd, 1), shift)
        else:
            room = torch.zeros(nkv * (n * hd + shift) + shift, dtype=dtype, device=DEV)
            view = room.as_strided((n, nkv, hd), (hd, n * hd + shift, 1), shift)
        view.copy_(x.to(DEV))
        put.append(view)
    cache, model = backend.kv8(nkv, hd, 2), Model(nkv, hd, 2)
    assert cache.append(Kv8Seqs(start=i32([0]), max_rows=n, max_blocks=2), *put)
    model.append(0, k.float().numpy(), v.float().numpy())
    for g, w in zip(read(cache, [0], [n], 2), model.values(n)):
        assert np.array_equal(g, w)


def test_a_pool_of_more_than_four_gigabytes(backend):
    nkv, hd = 8, 128
    n_blocks = (9 << 29) // ((64 * hd + 32) * nkv)  # 4.5 GB
    cache = backend.kv8(nkv, hd, n_blocks)
    assert cache.bytes() == (64 * hd + 32) * nkv * n_blocks > 1 << 32
    rng = np.random.default_rng(3)
    k, v = (rows_of(rng, 64, nkv, hd, torch.float16) for _ in range(2))
    for table in ([n_blocks - 1, 0], [n_blocks // 2, n_blocks - 2]):
        model = Model(nkv, hd, 2)
        assert cache.append(Kv8Seqs(start=i32([0]), max_rows=64, max_blocks=2, table=i32([table])), k.to(DEV), v.to(DEV))
        model.append(0, k.float().numpy(), v.float().numpy())
        for g, w in zip(read(cache, [0], [64], 2, i32([table])), model.values(64)):
            assert np.array_equal(g, w)
        k, v = v, k
    cache.free()


def test_arrays_that_do_not_fit_are_reported_and_touch_nothing_else(backend):
    nkv, hd, max_blocks = 2, 64, 2
    rng = np.random.default_rng(4)
    k, v = (rows_of(rng, 6, nkv, hd, torch.float32).to(DEV) for _ in range(2))

    def fresh():
        cache = backend.kv8(nkv, hd, 6)
        assert cache.append(Kv8Seqs(start=i32([0, 0, 0]), max_rows=2, max_blocks=max_blocks), k, v)
        return cache

    before = read(fresh(), [0, 0, 0], [2, 2, 2], max_blocks)
    good = dict(start=[2, 2, 2], rows=[0, 2, 4, 6], table=[[0, 1], [2, 3], [4, 5]])
    for left_out, bad in ((1, dict(start=[2, -1, 2])), (1, dict(start=[2, 63, 2])), (1, dict(start=[2, 2 ** 31 - 1, 2])), (1, dict(rows=[0, 2, 1, 6])),
                          (0, dict(rows=[-1, 2, 4, 6])), (2, dict(rows=[0, 2, 4, 7])), (1, dict(table=[[0, 1], [6, 3], [4, 5]])),
                          (1, dict(table=[[0, 1], [-1, 3], [4, 5]]))):
        cache, a = fresh(), {**good, **bad}
        seqs = Kv8Seqs(start=i32(a["start"]), rows=i32(a["rows"]), n_rows=6, max_rows=2, max_blocks=max_blocks, table=i32(a["table"]))
        assert cache.append(seqs, k, v)
        torch.cuda.synchronize()
        with pytest.raises(ob.BackendError) as e:
            backend.check_status()
        assert e.value.code == -2 and "8-bit cache" in str(e.value)
        backend.check_status()  # (reported once)
        whole = read(cache, [0, 0, 0], [4, 2, 4] if left_out == 1 else [2, 4, 4] if left_out == 0 else [4, 4, 2], max_blocks)
        assert all(np.isfinite(x).all() for x in whole)
        for g, w in zip(read(cache, [0, 0, 0], [2, 2, 2], max_blocks), before):
            assert np.array_equal(g[2 * left_out:2 * left_out + 2], w[2 * left_out:2 * left_out + 2]), bad


def test_refusals(backend):
    assert backend.kv8(2, 96, 4) is None and "head dimension" in backend.last_declined
    assert backend.kv8(5000, 64, 4) is None
    for nkv, hd, blocks in ((0, 64, 4), (2, 64, 0)):
        with pytest.raises(ob.BackendError):
            backend.kv8(nkv, hd, blocks)
    cache = backend.kv8(2, 64, 4)
    k = torch.zeros((4, 2, 64), device=DEV)
    start = i32([0])
    for seqs in (Kv8Seqs(start=start, max_rows=4, max_blocks=5),              # more blocks than the pool has, without a table
                 Kv8Seqs(start=start, max_rows=4, max_blocks=0),
                 Kv8Seqs(start=start, max_rows=0, max_blocks=4, rows=i32([0, 4]), n_rows=4),
                 Kv8Seqs(start=start, max_rows=5, max_blocks=4, rows=i32([0, 4]), n_rows=4)):
        with pytest.raises(ob.BackendError) as e:
            cache.append(seqs, k, k)
        assert e.value.code == -2
    none = k[:0]
    assert cache.append(Kv8Seqs(start=start, rows=i32([0, 0]), n_rows=0, max_rows=0, max_blocks=4), none, none)  # nothing to do
    assert cache.append(Kv8Seqs(start=i32([]), max_rows=1, max_blocks=4), none, none)
    L = ob.lib()
    import ctypes as C

    s = Kv8Seqs(start=start, max_rows=4, max_blocks=4).c(k.device)
    assert L.b2_kv8_append_dev(backend._ctx, cache.handle, C.byref(s), k.data_ptr(), k.data_ptr(), 9, 128, 64) == -2
    assert L.b2_kv8_append_dev(backend._ctx, cache.handle, C.byref(s), None, k.data_ptr(), 0, 128, 64) == -2
    assert L.b2_kv8_append_dev(backend._ctx, cache.handle, None, k.data_ptr(), k.data_ptr(), 0, 128, 64) == -2
    assert L.b2_kv8_append_dev(backend._ctx, 1 << 40, C.byref(s), k.data_ptr(), k.data_ptr(), 0, 128, 64) == -2
    assert L.b2_kv8_read_dev(backend._ctx, cache.handle, C.byref(s), k.data_ptr() + 4, k.data_ptr()) == -2
    assert L.b2_kv8_free(backend._ctx, 1 << 40) == -2 and L.b2_kv8_bytes(backend._ctx, 1 << 40) == 0
