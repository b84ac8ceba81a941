"""Attention of few rows over long contexts in the 8-bit cache, whose blocks are dealt out over all of the GPU, and the bounds of a call."""
import ctypes as C
import math

import pytest
import torch

import oxinfer_b200 as ob
from oxinfer_b200.kv8 import Kv8Seqs

from test_attend_kv8_gpu import DEV, Setting, i32, slopes_of

pytestmark = pytest.mark.gpu

RAGGED = [3000, 1, 2999, 31, 64, 2017, 33, 2800, 700, 32, 1500, 2999, 95, 65, 2500, 3000]


def dealt(backend, s, **kw):
    """The check, and that it took two launches: the attention and the sums of what its CTAs share."""
    before = backend.launch_count()
    out = s.check(**kw)
    assert backend.launch_count() - before == 2
    return out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(8, 8), (32, 8), (20, 4)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_ragged_sequences(backend, nh, nkv, hd, dtype):
    dealt(backend, Setting(backend, RAGGED * (2 if nkv == 4 else 1), [1] * len(RAGGED) * (2 if nkv == 4 else 1), nh, nkv, hd, dtype, seed=nh + hd, spread=2.0))


def test_sequences_without_rows_and_with_several(backend):
    counts = [0, 1, 3, 0, 5, 1, 0, 2, 1, 7, 0, 1, 1, 2, 0, 0]
    s = Setting(backend, [max(n, c) for n, c in zip(RAGGED, counts)], counts, 8, 8, 64, "f32", seed=20)
    dealt(backend, s)
    dealt(backend, s, prefix=[(37 * i * i) % 3000 for i in range(16)], slopes=slopes_of(8), cap=20.0)
    dealt(backend, s, prefix=[(37 * i * i) % 3000 for i in range(16)], window=70)


@pytest.mark.parametrize("lengths,counts,nh,nkv", [([20000], [1], 8, 8), ([17001], [2], 32, 8), ([9000, 50, 1, 8200], [1, 1, 1, 1], 4, 4), ([9000, 50, 300, 8200], [0, 3, 8, 1], 4, 4),
                                                   ([40001], [1], 2, 1)])
@pytest.mark.parametrize("hd", [64, 128])
def test_few_units(backend, lengths, counts, nh, nkv, hd):
    """A unit's blocks over many CTAs."""
    s = Setting(backend, lengths, counts, nh, nkv, hd, "f32", seed=sum(lengths), spread=2.0)
    dealt(backend, s)
    dealt(backend, s, cap=15.0, slopes=slopes_of(nh))


def test_values_that_are_not_finite(backend):
    poison = [(0, 5, 2, 0), (2, 2998, 1, 1), (5, 2000, 3, 1), (15, 2900, 0, 0)]
    counts = [1] * 15 + [200]
    s = Setting(backend, RAGGED, counts, 8, 8, 64, "f32", seed=21, poison=poison)
    out = s.check()
    assert 0 < int(torch.isnan(out).any(-1).sum()) < out.shape[0] * 8
    s = Setting(backend, RAGGED, [1] * 16, 8, 8, 64, "f32", seed=22, poison=poison)
    out = dealt(backend, s)
    assert int(torch.isnan(out).any(-1).sum()) == 4
    s.q[3, 2, 7] = math.inf
    again = torch.empty_like(s.q)
    assert s.cache.attend(s.seqs, s.q, again, scale=s.scale)
    assert torch.isnan(again[3, 2]).all()
    again[3, 2] = out[3, 2]
    assert torch.equal(again.nan_to_num(7.0), out.nan_to_num(7.0))


def test_with_and_without_memory_of_its_own(backend):
    s = Setting(backend, [20000], [1], 8, 2, 64, "f32", seed=23)
    y, tol = s.want()
    L, cs = ob.lib(), s.seqs.c()
    work = torch.full((L.b2_attend_kv8_work_bytes(backend._ctx, s.cache.handle) + 16,), 255, dtype=torch.uint8, device=DEV)  # (NaN everywhere)
    for at, launches in ((None, 1), (work.data_ptr(), 2)):
        out, before = torch.full_like(s.q, 9.0), backend.launch_count()
        a = ob._lib.Kv8Attention(8, s.scale, 0.0, 0, None, None, at)
        assert L.b2_attend_kv8_dev(backend._ctx, s.cache.handle, C.byref(cs), C.byref(a), s.q.data_ptr(), 512, out.data_ptr(), 512, 0) == 0
        assert ((out.double() - y).abs() <= tol).all() and backend.launch_count() - before == launches
    assert (work[-16:] == 255).all()
    a = ob._lib.Kv8Attention(8, s.scale, 0.0, 0, None, None, work.data_ptr() + 8)
    assert L.b2_attend_kv8_dev(backend._ctx, s.cache.handle, C.byref(cs), C.byref(a), s.q.data_ptr(), 512, out.data_ptr(), 512, 0) == -2


def test_memory_is_the_backends_streams(backend):
    """The sums' memory may be handed on only behind the launch: torch's allocator goes by stream."""
    cache, side = backend.kv8(2, 64, 4), torch.cuda.Stream()
    n = cache._work_bytes
    torch.cuda.synchronize()
    backend.set_stream(side.cuda_stream)
    try:
        work = cache._work()
        at = work.data_ptr()
        del work
        assert torch.empty(n, dtype=torch.uint8, device=DEV).data_ptr() != at
        with torch.cuda.stream(side):
            assert cache._work().data_ptr() == at
    finally:
        backend.set_stream(0)


def test_two_streams_at_once_and_captured(backend):
    s = Setting(backend, [30000], [1], 8, 2, 128, "f32", seed=24)
    want = dealt(backend, s)
    other = ob.Backend(0)
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [torch.empty((20,) + tuple(s.q.shape), device=DEV) for _ in sides]
    torch.cuda.synchronize()
    t = Setting(other, [30000], [1], 8, 2, 128, "f32", seed=24)
    torch.cuda.synchronize()
    backend.set_stream(sides[0].cuda_stream), other.set_stream(sides[1].cuda_stream)
    try:
        for i in range(20):
            for x, out in ((s, outs[0]), (t, outs[1])):
                assert x.cache.attend(x.seqs, x.q, out[i], scale=x.scale)
        torch.cuda.synchronize()
        for out in outs:
            assert all(torch.equal(out[i], want) for i in range(20))
        graphs = []
        for x, out, side in ((s, outs[0], sides[0]), (t, outs[1], sides[1])):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                assert x.cache.attend(x.seqs, x.q, out[0], scale=x.scale)
            graphs.append(graph)
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for _ in range(20):
            for graph, side in zip(graphs, sides):
                with torch.cuda.stream(side):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out[0], want) for out in outs)
    finally:
        torch.cuda.synchronize()
        backend.set_stream(0)
        t.cache.free()
        other.close()
    backend.check_status()


def test_sequences_that_share_blocks(backend):
    """A prefix that two sequences have in common, read where it lies."""
    s = Setting(backend, [3000, 2000], [1, 1], 16, 8, 64, "f32", seed=25)
    table = s.table.clone()
    table[1] = table[0]
    seqs = Kv8Seqs(start=i32([2999, 2999]), max_blocks=s.max_blocks, table=table)
    q, out = s.q[:1].expand(2, -1, -1).contiguous(), torch.empty_like(s.q)
    assert s.cache.attend(seqs, q, out, scale=s.scale)
    y, tol = s.want()
    assert all(((out[i].double() - y[0]).abs() <= tol[0]).all() for i in range(2))


@pytest.mark.parametrize("dtype,count", [("f32", 1), ("bf16", 40)])
def test_blocks_beyond_four_gigabytes(backend, dtype, count):
    """The last blocks of a large pool: offsets that 32 bits do not hold."""
    n_blocks, used = 66000, 100
    big = backend.kv8(8, 128, n_blocks)
    assert big.bytes() > 1 << 32
    s = Setting(backend, [used * 32 - 5], [count], 16, 8, 128, dtype, seed=26)
    want = s.check()
    table = i32([[n_blocks - 1 - i for i in range(used)]])
    n = used * 32 - 5
    assert big.append(Kv8Seqs(start=i32([0]), max_blocks=used, max_rows=n, table=table), s.k, s.v)  # (what a cache stands for is kept as it is)
    k, v = torch.empty_like(s.k), torch.empty_like(s.v)
    assert big.read(Kv8Seqs(start=i32([0]), max_blocks=used, max_rows=n, table=table), k, v) and torch.equal(k, s.k) and torch.equal(v, s.v)
    out = torch.empty_like(s.q)
    assert big.attend(Kv8Seqs(start=s.seqs.start, max_blocks=used, max_rows=count, table=table), s.q, out, scale=s.scale)
    assert torch.equal(out, want)
    big.free()


def test_heads_beyond_the_tcgen05_forms_arithmetic(backend):
    """Rows times heads a KV head squared past 2^31: the other form takes them."""
    G, t, n = 2048, 513, 600
    s = Setting(backend, [n], [t], 4, 1, 64, "f16", seed=27)
    y, tol = s.want()
    q = s.q.repeat(1, G // 4, 1)
    out = torch.empty_like(q)
    assert s.cache.attend(s.seqs, q, out, scale=s.scale)
    got = out.view(t, G // 4, 4, 64)
    assert torch.equal(got, got[:, :1].expand_as(got))
    assert ((got[:, 0].double() - y).abs() <= tol).all()


def test_bounds_of_a_call(backend):
    s = Setting(backend, [40], [1], 4, 2, 64, "f32", seed=28)
    out = torch.full_like(s.q, 3.0)
    for kw in (dict(scale=2.0 ** 61), dict(scale=-(2.0 ** 61)), dict(scale=math.inf), dict(scale=1.0, cap=2.0 ** 61), dict(scale=1.0, cap=2.0 ** -61)):
        with pytest.raises(ob.BackendError) as e:
            s.cache.attend(s.seqs, s.q, out, **kw)
        assert e.value.code == -2
    assert (out == 3.0).all()
    for cap in (2.0 ** 60, 2.0 ** 40):  # (far above the scores: as without one)
        s.check()
        assert s.cache.attend(s.seqs, s.q, out, scale=s.scale, cap=cap)
        y, tol = s.want()
        assert ((out.double() - y).abs() <= tol).all()
    # more sequences than a call takes: declined before anything is looked at
    L, start = ob.lib(), s.seqs.start
    n = (1 << 25) + 1
    cs = ob._lib.Kv8Seqs(n, n, 1, 1, start.data_ptr(), start.data_ptr(), None)
    a = ob._lib.Kv8Attention(4, 1.0, 0.0, 0, None, None, None)
    before = backend.launch_count()
    assert L.b2_attend_kv8_dev(backend._ctx, s.cache.handle, C.byref(cs), C.byref(a), s.q.data_ptr(), 256, out.data_ptr(), 256, 0) == ob.DECLINED
    assert L.b2_kv8_append_dev(backend._ctx, s.cache.handle, C.byref(cs), s.q.data_ptr(), s.q.data_ptr(), 0, 0, 64) == ob.DECLINED
    assert L.b2_kv8_read_dev(backend._ctx, s.cache.handle, C.byref(cs), out.data_ptr(), out.data_ptr()) == ob.DECLINED
    assert backend.launch_count() == before
