"""Attention over the 8-bit cache (b2_attend_kv8_dev) against the formula in 64 bits over the values that the cache stands for."""
import math

import numpy as np
import pytest
import torch

import oxinfer_b200 as ob
from oxinfer_b200.kv8 import BLOCK, Kv8Seqs

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


class Setting:
    """Sequences of given lengths in a pool with shuffled blocks; their last `counts` tokens are the call's queries."""

    def __init__(self, backend, lengths, counts, nh, nkv, hd, dtype, seed, spread=1.0, poison=()):
        self.be, self.lengths, self.counts, self.nh, self.nkv, self.hd, self.dtype = backend, lengths, counts, nh, nkv, hd, TYPES[dtype]
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        rng = np.random.default_rng(seed)
        n_seqs = len(lengths)
        self.max_blocks = max(1, max(-(-n // BLOCK) for n in lengths))
        self.table = i32(rng.permutation(n_seqs * self.max_blocks + 2)[:n_seqs * self.max_blocks].reshape(n_seqs, -1))
        self.cache = backend.kv8(nkv, hd, n_seqs * self.max_blocks + 2)
        n = sum(lengths)
        k, v = (torch.randn((n, nkv, hd), device=DEV, generator=g) * s for s in (spread, 0.7))
        self.first_of = np.concatenate([[0], np.cumsum(lengths)])
        for seq, pos, head, kind in poison:
            (k, v)[kind][self.first_of[seq] + pos, head, 3] = math.nan
        every = Kv8Seqs(start=i32([0] * n_seqs), rows=i32(self.first_of), n_rows=n, max_rows=max(lengths), max_blocks=self.max_blocks, table=self.table)
        assert self.cache.append(every, k, v)
        self.k, self.v = torch.empty_like(k), torch.empty_like(v)
        assert self.cache.read(every, self.k, self.v)
        self.first = np.concatenate([[0], np.cumsum(counts)])
        self.n_rows = int(self.first[-1])
        self.seqs = Kv8Seqs(start=i32([a - b for a, b in zip(lengths, counts)]), rows=i32(self.first), n_rows=self.n_rows, max_rows=max(1, max(counts)),
                            max_blocks=self.max_blocks, table=self.table)
        self.q = (torch.randn((self.n_rows, nh, hd), device=DEV, generator=g) * 1.5).to(self.dtype)
        self.scale = 1.0 / math.sqrt(hd)

    def want(self, cap=0.0, window=0, slopes=None, prefix=None):
        """The formula in 64 bits, and how far a result may be off.

        Bound: queries and probabilities in two f16 terms are off by 2^-22 of them, a sum of HD products in HD / 16 + 3 steps of at most 2^-23 of the sum of
        magnitudes A each: a score is off by less than (2^-22 + 11 * 2^-23) A < 2^-19.6 A (the cap's slope is at most one), by 2^-22 of a cap and 2^-23 of a bias more; a
        probability by twice that, 2^-21 for the exponentials and 2^-22 for its terms, the sums of n probabilities and of values by 2^-21 again: together
        2^-18.5 A + 2^-19 of the values' largest. One f16 term of the probabilities (16-bit results of more than eight rows a KV head): 2^-11 of it. A result's
        own rounding: half a step."""
        y = torch.zeros((self.n_rows, self.nh, self.hd), device=DEV, dtype=torch.float64)
        tol = torch.zeros((self.n_rows, self.nh, 1), device=DEV, dtype=torch.float64)
        G = self.nh // self.nkv
        few = self.dtype == torch.float32 or max(self.counts) * G <= 8
        for s, (n, t) in enumerate(zip(self.lengths, self.counts)):
            if t == 0:
                continue
            k, v = (x[self.first_of[s]:self.first_of[s + 1]].double() for x in (self.k, self.v))
            j, p = torch.arange(n, device=DEV), torch.arange(n - t, n, device=DEV)
            see = j[None] <= p[:, None]
            if prefix is not None:
                see |= j[None] < prefix[s]
            if window:
                see &= p[:, None] - j[None] < window
            for h in range(self.nh):
                q = self.q[self.first[s]:self.first[s + 1], h].double()
                sc = q @ k[:, h // G].T * self.scale
                a = (q.abs() @ k[:, h // G].abs().nan_to_num(0.0).T * abs(self.scale)).amax(1, keepdim=True)
                if cap:
                    sc = cap * torch.tanh(sc / cap)
                if slopes is not None:
                    sc = sc + slopes[h].double() * (j[None] - p[:, None])
                sc = torch.where(see, sc, -math.inf)
                w = torch.softmax(sc, -1)
                o = w @ v[:, h // G].nan_to_num(0.0)
                lost = (torch.isnan(sc) | torch.isnan(v[:, h // G]).any(1)[None]) & see  # (what is not seen is nobody's)
                o[lost.any(1)] = math.nan
                y[self.first[s]:self.first[s + 1], h] = o
                vmax = v[:, h // G].nan_to_num(0.0).abs().amax()
                bias = slopes[h].abs().double() * n if slopes is not None else 0.0
                d = vmax * (2.0 ** -18.5 * a + 2.0 ** -19 + cap * 2.0 ** -20 + bias * 2.0 ** -21 + (0.0 if few else 2.0 ** -11))
                tol[self.first[s]:self.first[s + 1], h] = d
        if self.dtype != torch.float32:
            tol = tol + torch.finfo(self.dtype).eps / 2 * (y.abs().nan_to_num(0.0) + tol)
        return y, tol

    def check(self, **kw):
        y, tol = self.want(**{k: v for k, v in kw.items()})
        out = torch.full_like(self.q, 9.0)
        pre = i32(kw["prefix"]) if kw.get("prefix") is not None else None
        assert self.cache.attend(self.seqs, self.q, out, scale=self.scale, cap=kw.get("cap", 0.0), window=kw.get("window", 0), slopes=kw.get("slopes"), prefix=pre)
        torch.cuda.synchronize()
        self.be.check_status()
        got = out.double()
        assert torch.equal(torch.isnan(got), torch.isnan(y))
        err = ((got - y).abs() - tol).nan_to_num(0.0)
        assert (err <= 0).all(), (float((got - y).abs().nan_to_num(0.0).max()), float(err.max()))
        return out


def slopes_of(nh):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / nh) for i in range(nh)], device=DEV)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(4, 4), (8, 2), (8, 1), (6, 2), (20, 1)])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_one_token_of_every_length(backend, nh, nkv, hd, dtype):
    Setting(backend, [1, 2, 31, 32, 33, 63, 64, 65, 200, 1000], [1] * 10, nh, nkv, hd, dtype, seed=nh * hd).check()


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("counts", [[1, 0, 2, 5], [4, 4, 4, 4], [17, 3, 0, 40], [70, 33, 64, 1]])
@pytest.mark.parametrize("nh,nkv,hd", [(4, 1, 128), (3, 3, 64), (16, 2, 64)])
def test_several_tokens_of_ragged_sequences(backend, nh, nkv, hd, counts, dtype):
    Setting(backend, [c + e for c, e in zip(counts, (0, 45, 700, 31))], counts, nh, nkv, hd, dtype, seed=sum(counts)).check()


@pytest.mark.parametrize("kw", [dict(window=1), dict(window=33), dict(window=64, cap=20.0), dict(window=2 ** 32 - 1), dict(cap=0.5), dict(cap=50.0), dict(prefix=[3, 40, 0]),
                                dict(prefix=[500, 1, 33], window=40), dict(slopes=True), dict(slopes=True, cap=30.0, window=100, prefix=[0, 90, 20])], ids=str)
@pytest.mark.parametrize("counts", [[1, 1, 1], [9, 50, 2]])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_caps_biases_windows_and_prefixes(backend, kw, counts, dtype):
    kw = dict(kw)
    if "slopes" in kw:
        kw["slopes"] = slopes_of(8)
    Setting(backend, [70, 300, 129], counts, 8, 2, 128, dtype, seed=77, spread=3.0).check(**kw)


@pytest.mark.parametrize("nkv,length", [(1, 20000), (4, 9000), (8, 2049)])
def test_long_contexts_of_one_sequence(backend, nkv, length):
    """Clusters of every size share a sequence's keys."""
    Setting(backend, [length], [1], 4 * nkv, nkv, 128, "f32", seed=length, spread=2.0).check()
    Setting(backend, [length], [3], 4 * nkv, nkv, 64, "f32", seed=length, spread=2.0).check()


def test_scores_far_apart_and_magnitudes_far_from_one(backend):
    for spread, qs in ((40.0, 30.0), (1e-18, 1e18), (1e18, 1e-18), (1e-3, 1e-3)):
        s = Setting(backend, [100, 333], [1, 20], 4, 2, 64, "f32", seed=5, spread=spread)
        s.q *= qs
        s.check()


def test_a_value_that_is_not_finite_reaches_the_rows_that_see_it_and_no_others(backend):
    """Keys (kind 0) and values (kind 1) that are NaN: in sight of all rows, of the later ones, out of the window, and behind a row."""
    for dtype in ("f32", "f16"):
        for kind in (0, 1):
            s = Setting(backend, [90, 150, 64], [12, 40, 1], 4, 2, 64, dtype, seed=6, poison=[(0, 85, 1, kind), (1, 20, 0, kind), (2, 3, 0, kind)])
            out = s.check(window=50)
            assert torch.isnan(out[7:12, 2:]).all() and not torch.isnan(out[:7]).any() and not torch.isnan(out[7:12, :2]).any()
            assert not torch.isnan(out[12:]).any()  # (out of the window)
            assert torch.isnan(s.check()[52:, :2]).all()


def test_queries_that_are_not_finite_reach_their_own_rows(backend):
    s = Setting(backend, [60, 90], [1, 9], 4, 2, 128, "f32", seed=9)
    clean = s.check()
    s.q[3, 1, 100] = math.inf
    s.q[0, 2, 0] = math.nan
    out = torch.empty_like(s.q)
    assert s.cache.attend(s.seqs, s.q, out, scale=s.scale)
    hit = torch.zeros((10, 4), dtype=torch.bool, device=DEV)
    hit[3, 1] = hit[0, 2] = True
    assert torch.isnan(out[hit]).all() and torch.equal(out[~hit], clean[~hit])


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides_alignments_and_results_in_place(backend, dtype, shift):
    s = Setting(backend, [40, 77], [3, 5], 4, 2, 64, dtype, seed=12)
    want = s.check()
    width = 4 * 64 + 16 + shift
    room = torch.full((9 * width + shift,), 5.0, dtype=s.dtype, device=DEV)
    rows = room.as_strided((8, 4, 64), (width, 64, 1), shift)
    rows.copy_(s.q)
    assert s.cache.attend(s.seqs, rows, rows, scale=s.scale)  # over the queries themselves
    assert torch.equal(rows, want)
    left = torch.ones_like(room, dtype=torch.bool)
    left.as_strided((8, 4, 64), (width, 64, 1), shift).fill_(False)
    assert (room[left] == 5.0).all()  # between the rows, and behind the last


def test_rows_that_no_sequence_has_stay_as_they_were(backend):
    s = Setting(backend, [40, 77], [3, 5], 4, 2, 64, "f32", seed=13)
    want = s.check()
    q = torch.cat([s.q, s.q[:4]])
    out = torch.full_like(q, 4.0)
    seqs = Kv8Seqs(start=s.seqs.start, rows=s.seqs.rows, n_rows=12, max_rows=2, max_blocks=s.max_blocks, table=s.table)  # (and a hint below the longest)
    assert s.cache.attend(seqs, q, out, scale=s.scale)
    assert (out[8:] == 4.0).all() and torch.allclose(out[:8], want, rtol=0, atol=1e-5)


def test_streams_and_captured_steps(backend):
    """A captured step (append, attend) replayed as its positions move on, two graphs of one cache, on a stream of their own."""
    nh, nkv, hd, n_seqs, max_blocks = 8, 2, 64, 3, 4
    g = torch.Generator(device=DEV)
    g.manual_seed(3)
    total = 50
    k, v = (torch.randn((total, n_seqs, nkv, hd), device=DEV, generator=g) for _ in range(2))
    q = torch.randn((total, n_seqs, nh, hd), device=DEV, generator=g)
    eager = backend.kv8(nkv, hd, n_seqs * max_blocks)
    want = []
    for i in range(total):
        seqs = Kv8Seqs(start=i32([i] * n_seqs), max_blocks=max_blocks)
        out = torch.empty_like(q[0])
        assert eager.append(seqs, k[i], v[i]) and eager.attend(seqs, q[i], out, scale=0.125)
        want.append(out)
    side = torch.cuda.Stream()
    cache = backend.kv8(nkv, hd, n_seqs * max_blocks)
    start, kb, vb, qb, ob_ = i32([0] * n_seqs), k[0].clone(), v[0].clone(), q[0].clone(), torch.empty_like(q[0])
    seqs = Kv8Seqs(start=start, max_blocks=max_blocks)
    torch.cuda.synchronize()
    backend.set_stream(side.cuda_stream)
    try:
        graphs = []
        for part in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=side):
                if part == 0:
                    assert cache.append(seqs, kb, vb)
                else:
                    assert cache.attend(seqs, qb, ob_, scale=0.125)
            graphs.append(graph)
        with torch.cuda.stream(side):
            for i in range(total):
                start.fill_(i)
                kb.copy_(k[i]), vb.copy_(v[i]), qb.copy_(q[i])
                for graph in graphs:
                    graph.replay()
                assert torch.equal(ob_, want[i]), i
    finally:
        torch.cuda.synchronize()
        backend.set_stream(0)
    backend.check_status()


def test_arrays_that_do_not_fit_are_reported(backend):
    s = Setting(backend, [40, 77], [1, 1], 4, 2, 64, "f32", seed=14)
    want = s.check()
    table = s.table.clone()
    table[0, 0] = 1 << 20
    for bad in (dict(start=i32([39, 5000])), dict(start=i32([-1, 76])), dict(rows=i32([0, 1, 9])), dict(table=table)):
        a = dict(start=s.seqs.start, rows=s.seqs.rows, n_rows=2, max_rows=1, max_blocks=s.max_blocks, table=s.table)
        out = torch.full_like(s.q, 3.0)
        assert s.cache.attend(Kv8Seqs(**{**a, **bad}), s.q, out, scale=s.scale)
        torch.cuda.synchronize()
        with pytest.raises(ob.BackendError) as e:
            backend.check_status()
        assert e.value.code == -2
        ok = 1 if ("table" in bad or (bad.get("start") is not None and int(bad["start"][0]) == -1)) else 0
        assert torch.equal(out[ok], want[ok]), bad  # the other sequence's


def test_refusals(backend):
    import ctypes as C

    s = Setting(backend, [40], [1], 4, 2, 64, "f32", seed=15)
    out = torch.empty_like(s.q)
    for kw in (dict(scale=math.nan), dict(scale=1.0, cap=-1.0), dict(scale=1.0, cap=math.inf)):
        with pytest.raises(ob.BackendError) as e:
            s.cache.attend(s.seqs, s.q, out, **kw)
        assert e.value.code == -2
    with pytest.raises(ob.BackendError):
        s.cache.attend(s.seqs, s.q[:, :3], out[:, :3], scale=1.0)  # three heads over two
    L, cs = ob.lib(), s.seqs.c(s.q.device)
    a = ob._lib.Kv8Attention(4, 1.0, 0.0, 0, None, None, None)
    args = lambda **k: [backend._ctx, s.cache.handle, C.byref(cs), C.byref(a), s.q.data_ptr(), 256, out.data_ptr(), 256, 0]
    for i, bad in ((1, 1 << 40), (2, None), (3, None), (4, None), (6, None), (8, 7)):
        x = args()
        x[i] = bad
        assert L.b2_attend_kv8_dev(*x) == -2, i
    two = Setting(backend, [40, 50], [1, 1], 4, 2, 64, "f32", seed=16)
    cs = two.seqs.c(s.q.device)
    assert L.b2_attend_kv8_dev(backend._ctx, two.cache.handle, C.byref(cs), C.byref(a), two.q.data_ptr(), 256, two.q.data_ptr(), 255, 0) == -2
