"""Calls of the 8-bit cache and of rules on logits that their documentation allows: strides, alignments, results over inputs, sizes of one and of none."""
import ctypes as C

import pytest
import torch

import oxinfer_b200 as ob
from oxinfer_b200.kv8 import Kv8Seqs

from test_attend_kv8_gpu import DEV, Setting, i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,nkv", [(1, 1), (1, 3), (5, 1)])
def test_strides_of_dimensions_of_one_mean_nothing(backend, rows, nkv):
    hd = 64
    k, v, q = (torch.randn((rows, nkv, hd), device=DEV) for _ in range(3))

    def odd(x, a, b):
        return x.as_strided(x.shape, (a if rows == 1 else nkv * hd, b if nkv == 1 else hd, 1))

    seqs = Kv8Seqs(start=i32([0]), max_rows=rows, max_blocks=1)
    one, two = backend.kv8(nkv, hd, 1), backend.kv8(nkv, hd, 1)
    assert one.append(seqs, k, v) and two.append(seqs, odd(k, 7, 1000003), odd(v, 1 << 40, 3))
    a, b = (torch.empty((2, rows, nkv, hd), device=DEV) for _ in range(2))
    assert one.read(seqs, a[0], a[1]) and two.read(seqs, b[0], b[1]) and torch.equal(a, b)
    x, y = torch.empty_like(q), torch.empty_like(q)
    assert one.attend(seqs, q, x, scale=0.125) and two.attend(seqs, odd(q, 0, 5), odd(y, 1, 0), scale=0.125) and torch.equal(x, y)


def test_rows_of_one_logit(backend):
    room = torch.tensor([[3.0, 9.0], [-2.0, 9.0], [float("nan"), 9.0]], device=DEV)
    x, out, pick = room[:, :1], torch.full((3, 5), 7.0, device=DEV), torch.full((3,), -9, dtype=torch.int32, device=DEV)
    assert x.stride() == (2, 1)
    for view in (x, x.as_strided((3, 1), (2, 17))):
        assert backend.logits_dev(view, out.as_strided((3, 1), (5, 3)), pick) and pick.tolist() == [0, 0, -1]
        assert torch.equal(out[:2, 0], x[:2, 0]) and torch.isnan(out[2, 0]) and (out[:, 1:] == 7.0).all()


def test_results_over_other_rows_are_refused(backend):
    """The input's own rows, rows beside them and rows behind them are fine."""
    s = Setting(backend, [40, 77], [3, 5], 4, 2, 64, "f16", seed=41)
    want, w = s.check(), 4 * 64
    for q_at, qs, o_at, os, fine in ((0, w, 0, w, True), (0, 2 * w, w, 2 * w, True), (w, 2 * w, 0, 2 * w, True), (0, 2 * w + 8, w + 8, 2 * w + 8, True), (0, w, 8 * w, w, True),
                                     (8 * 2 * w, w, 0, 2 * w, True), (0, 2 * w, 3 * w, 2 * w, True),
                                     (0, 2 * w, 0, w, False), (0, w, 0, 2 * w, False), (0, w, w, w, False), (w, w, 0, w, False), (0, 2 * w, w - 1, 2 * w, False), (0, 2 * w, w + 1, 2 * w, False),
                                     (0, 2 * w, 2 * w, 2 * w, False), (0, w, 7 * w, w, False)):
        room = torch.full((30 * w,), 5.0, dtype=s.dtype, device=DEV)
        q, out = (room.as_strided((8, 4, 64), (stride, 64, 1), at) for at, stride in ((q_at, qs), (o_at, os)))
        q.copy_(s.q)
        before = room.clone()
        if fine:
            assert s.cache.attend(s.seqs, q, out, scale=s.scale) and torch.equal(out, want), (q_at, qs, o_at, os)
            continue
        with pytest.raises(ob.BackendError) as e:
            s.cache.attend(s.seqs, q, out, scale=s.scale)
        assert e.value.code == -2 and torch.equal(room, before), (q_at, qs, o_at, os)
    t, n = 6, 1000
    x = torch.randn((t, n), device=DEV)
    for x_at, xs, o_at, os, fine in ((0, n, 0, n, True), (0, 2 * n, n, 2 * n, True), (n, n, n + t * n, n, True), (0, 2 * n, 0, n, False), (0, n, 0, 2 * n, False), (0, n, n, n, False),
                                     (0, 2 * n, 2 * n - 1, 2 * n, False), (5, n, 0, n, False)):
        room = torch.full((3 * t * n,), 5.0, device=DEV)
        a, out = (room.as_strided((t, n), (stride, 1), at) for at, stride in ((x_at, xs), (o_at, os)))
        a.copy_(x)
        before = room.clone()
        if fine:
            assert backend.logits_dev(a, out) and torch.equal(out, x)
            continue
        with pytest.raises(ob.BackendError) as e:
            backend.logits_dev(a, out)
        assert e.value.code == -2 and torch.equal(room, before)
    one = torch.randn((1, n), device=DEV)  # (a row's stride means nothing)
    assert backend.logits_dev(one, one.as_strided((1, n), (3, 1)))


def test_rows_of_no_logits(backend):
    x, pick = torch.empty((3, 0), device=DEV), torch.full((3,), 7, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(x, x, pick) and pick.tolist() == [-1, -1, -1]
    assert backend.logits_dev(x, x) and backend.logits_dev(x[:0], None, pick[:0])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_of_logits_under_the_rules_of_several(backend, dtype):
    """A row that is read for all (stride zero), and rows that share a part of theirs; not over themselves."""
    t, n = 5, 20000
    room = torch.randn(n + 4 * 8, device=DEV).to(dtype)
    rules = ob.LogitRules(bias_ids=i32([11, 12, 13, 14, 15]), bias=torch.full((5,), 50.0, device=DEV), bias_ptr=i32([0, 1, 2, 3, 4, 5]))
    for stride in (0, 8):
        x, out, pick = room.as_strided((t, n), (stride, 1)), torch.empty((t, n), dtype=dtype, device=DEV), torch.empty(t, dtype=torch.int32, device=DEV)
        assert backend.logits_dev(x, out, pick, rules) and pick.tolist() == [11, 12, 13, 14, 15]
        want = x.float().clone()
        for i in range(t):
            want[i, 11 + i] += 50.0
        assert torch.equal(out, want.to(dtype))
        with pytest.raises(ob.BackendError):
            backend.logits_dev(x, x, pick, rules)


def test_addresses_between_elements_are_refused(backend):
    """Ahead of any launch."""
    s = Setting(backend, [40], [1], 4, 2, 64, "f32", seed=42)
    L, F32, F16 = ob.lib(), ob._lib.F32, ob._lib.F16
    room = torch.zeros(4096, device=DEV)
    at = room.data_ptr()
    words = i32([0, 1, 2, 3])
    w = words.data_ptr()
    seqs = lambda **k: C.byref(ob._lib.Kv8Seqs(**{**dict(n_seqs=1, n_rows=1, max_rows=1, max_blocks=1, table=None, start=w, rows=None), **k}))
    attn = lambda **k: C.byref(ob._lib.Kv8Attention(**{**dict(nh=4, scale=1.0, cap=0.0, window=0, slopes=None, prefix=None, work=None), **k}))
    rules = lambda **k: C.byref(ob._lib.LogitRules(**{**dict(repeat=1.5, frequency=0.0, presence=0.0), **k}))
    append = lambda q, k, v, t: L.b2_kv8_append_dev(backend._ctx, s.cache.handle, q, k, v, t, 128, 64)
    attend = lambda q, a, x, y, t: L.b2_attend_kv8_dev(backend._ctx, s.cache.handle, q, a, x, 256, y, 256, t)
    logits = lambda x, y, t, r, p: L.b2_logits_dev(backend._ctx, x, y, t, 1, 100, 100, 100, r, p)
    before = backend.launch_count()
    for rc in (append(seqs(), at + 2, at + 2048, F32), append(seqs(), at, at + 2049, F32), append(seqs(), at + 1, at, F16), append(seqs(start=w + 2), at, at, F32),
               append(seqs(table=w + 1), at, at, F32), append(seqs(rows=w + 2), at, at, F32), L.b2_kv8_read_dev(backend._ctx, s.cache.handle, seqs(start=w + 1), at, at + 2048),
               attend(seqs(), attn(), at + 2, at + 4096, F32), attend(seqs(), attn(), at, at + 4097, F16), attend(seqs(), attn(slopes=at + 2), at, at + 4096, F32),
               attend(seqs(), attn(prefix=w + 3), at, at + 4096, F32), attend(seqs(start=w + 2), attn(), at, at + 4096, F32),
               logits(at + 2, None, F32, None, w), logits(at, at + 4097, F16, None, w), logits(at, None, F32, None, w + 2), logits(at, None, F32, rules(n_history=1, history=w + 2), w),
               logits(at, None, F32, rules(n_history=1, history=w, history_ptr=w + 1), w), logits(at, None, F32, rules(n_bias=1, bias_ids=w + 2, bias=at), w),
               logits(at, None, F32, rules(n_bias=1, bias_ids=w, bias=at + 2), w), logits(at, None, F32, rules(n_bias=1, bias_ids=w, bias=at, bias_ptr=w + 2), w),
               logits(at, None, F32, rules(mask=w + 2), w)):
        assert rc == -2
    assert backend.launch_count() == before
    assert append(seqs(), at + 2, at + 514, F16) == 0 and attend(seqs(), attn(), at + 2, at + 4098, F16) == 0 and logits(at + 2, None, F16, None, w) == 0
    torch.cuda.synchronize()
    backend.check_status()


def test_windows_that_32_bits_do_not_hold(backend):
    for count in (1, 70):
        s = Setting(backend, [200], [count], 2, 1, 64, "f16", seed=43)
        want, out = s.check(), torch.empty_like(s.q)
        for window in (None, 0, 2 ** 32 - 1, 2 ** 32, 2 ** 32 + 7, 2 ** 40 + 1):
            assert s.cache.attend(s.seqs, s.q, out, scale=s.scale, window=window) and torch.equal(out, want), window
        with pytest.raises(AssertionError):
            s.cache.attend(s.seqs, s.q, out, scale=s.scale, window=-1)
