"""Rules on logits (b2_logits_dev) against the formulas, operation by operation."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import oxinfer_b200 as ob
from oxinfer_b200.sampling import LogitRules

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def i32(v):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)


def plain(x, rules, lists):
    """The rows as they are stored, and the choices. Single operations in f32 (numpy rounds each), then the type's rounding."""
    y = x.float().cpu().numpy().copy()
    t, n = y.shape
    f = np.float32
    for r in range(t):
        ids = [i for i in lists["history"][r] if 0 <= i < n]
        if (rules.repeat, rules.frequency, rules.presence) != (1.0, 0.0, 0.0):
            for i, c in zip(*np.unique(ids, return_counts=True)) if ids else []:
                l = y[r, i]
                l = l / f(rules.repeat) if l > 0 else l * f(rules.repeat)
                y[r, i] = l - (f(c) * f(rules.frequency) + f(rules.presence))
        last = {i: b for i, b in lists["bias"][r] if 0 <= i < n}
        for i, b in last.items():
            y[r, i] = y[r, i] + f(b)
        if lists["allowed"] is not None:
            y[r, ~lists["allowed"][r]] = -np.inf
    out = torch.from_numpy(y).to(x.dtype)
    s = out.float().numpy()
    pick = []
    for r in range(t):
        ok = np.where(s[r] > -np.inf)[0]
        pick.append(int(ok[np.argmax(s[r][ok])]) if len(ok) else -1)
    return out, pick


def words_of(allowed):
    t, n = allowed.shape
    bits = np.zeros((t, -(-n // 32) * 32), np.uint64)
    bits[:, :n] = allowed
    return (bits.reshape(t, -1, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32).view(np.int32)


def make(t, n, seed, history=0, biases=0, mask=None, **kw):
    rng = np.random.default_rng(seed)
    lists = {"history": [[] for _ in range(t)], "bias": [[] for _ in range(t)], "allowed": None}
    rules = dict(kw)
    if history:
        lists["history"] = [list(rng.integers(-2, min(n, 60) + 2, rng.integers(0, history + 1))) for _ in range(t)]  # (with ids outside, and repeated)
        rules.update(history=i32(sum(lists["history"], [])), history_ptr=i32(np.concatenate([[0], np.cumsum([len(h) for h in lists["history"]])])))
    if biases:
        lists["bias"] = [[(int(i), float(f)) for i, f in zip(rng.integers(-1, min(n, 90) + 1, m), rng.uniform(-4, 4, m).astype(np.float32))]
                         for m in rng.integers(0, biases + 1, t)]
        flat = sum(lists["bias"], [])
        rules.update(bias_ids=i32([i for i, _ in flat]), bias=torch.tensor([b for _, b in flat], dtype=torch.float32, device=DEV),
                     bias_ptr=i32(np.concatenate([[0], np.cumsum([len(b) for b in lists["bias"]])])))
    if mask is not None:
        lists["allowed"] = rng.random((t, n)) < mask
        rules.update(mask=torch.from_numpy(words_of(lists["allowed"])).to(DEV))
    return LogitRules(**rules), lists


def check(backend, x, rules, lists, out=None):
    want, pick = plain(x, rules, lists)
    out = torch.full_like(x, 3.0) if out is None else out
    got = torch.full((x.shape[0],), -9, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(x, out, got, rules)
    torch.cuda.synchronize()
    backend.check_status()
    assert np.array_equal(out.float().cpu().numpy(), want.float().numpy(), equal_nan=True)
    assert got.tolist() == pick


PENALTIES = dict(repeat=1.3, frequency=0.1, presence=0.7)


@pytest.mark.parametrize("n", [1, 3, 31, 32, 33, 8191, 8192, 8193, 128256, 131077])
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_every_rule_at_every_size(backend, n, dtype):
    g = torch.Generator(device=DEV)
    g.manual_seed(n)
    for t in (1, 5):
        x = (torch.randn((t, n), device=DEV, generator=g) * 3).to(TYPES[dtype])
        for kw in (dict(), dict(history=200, **PENALTIES), dict(biases=40), dict(mask=0.5), dict(mask=0.01), dict(history=300, biases=50, mask=0.9, **PENALTIES),
                   dict(history=100, repeat=0.5), dict(history=100, frequency=-0.4), dict(history=100)):
            check(backend, x, *make(t, n, n + t, **kw))


def test_vocabularies_of_more_than_a_cluster_counts_at_once(backend):
    x = torch.randn((2, 300001), device=DEV)
    rules, lists = make(2, 300001, 4, history=50, biases=50, mask=0.7, **PENALTIES)
    far = [131072, 262143, 300000, 300000, 7]
    lists["history"] = [far, far[::-1]]
    rules.history, rules.history_ptr = i32(far + far[::-1]), i32([0, 5, 10])
    check(backend, x, rules, lists)


@pytest.mark.parametrize("t,n,dtype,history,biases,mask", [(64, 70000, "f32", 900, 0, None), (40, 131077, "bf16", 0, 700, 0.5), (300, 32064, "bf16", 1500, 600, 0.6),
                                                            (150, 40000, "f16", 6000, 0, 0.3), (700, 9000, "f32", 100, 0, None), (620, 17000, "f16", 0, 0, 0.4), (30, 128256, "f32", 5000, 20, None)])
def test_many_rows_with_lists_all_over_them(backend, t, n, dtype, history, biases, mask):
    """Rows of several parts a CTA, lists of more tokens than a CTA's threads look at together, infinities and NaN among the logits; over the rows themselves, too."""
    rng = np.random.default_rng(t + n)
    x = torch.from_numpy((rng.standard_normal((t, n)) * 3).astype(np.float32))
    x[torch.from_numpy(rng.integers(0, t, 200)), torch.from_numpy(rng.integers(0, n, 200))] = math.nan
    x[torch.from_numpy(rng.integers(0, t, 50)), torch.from_numpy(rng.integers(0, n, 50))] = -math.inf
    x[t // 2, n - 2:] = math.inf
    x = x.to(TYPES[dtype]).to(DEV)
    rules, lists = make(t, n, t, mask=mask, **PENALTIES)
    if history:
        lists["history"] = [rng.integers(-3, n + 3, m).tolist() for m in rng.integers(0, history + 1, t)]
        lists["history"][0] = [n - 2] * history + [-1, n, n - 2]
        rules.history, rules.history_ptr = i32(sum(lists["history"], [])), i32(np.concatenate([[0], np.cumsum([len(h) for h in lists["history"]])]))
    if biases:
        lists["bias"] = [list(zip(rng.integers(-3, n + 3, m).tolist(), rng.uniform(-4, 4, m).astype(np.float32).tolist())) for m in rng.integers(0, biases + 1, t)]
        lists["bias"][t - 1] = [(n - 1, float(i)) for i in range(biases)]
        flat = sum(lists["bias"], [])
        rules.bias_ids, rules.bias = i32([i for i, _ in flat]), torch.tensor([b for _, b in flat], dtype=torch.float32, device=DEV)
        rules.bias_ptr = i32(np.concatenate([[0], np.cumsum([len(b) for b in lists["bias"]])]))
    check(backend, x, rules, lists)
    check(backend, x, rules, lists, out=x)


def test_ties_go_to_the_lower_token_and_nan_to_nobody(backend):
    x = torch.zeros((4, 70000), device=DEV)
    x[0, [40000, 9, 69999]] = 2.0
    x[1, 60001], x[1, 5] = math.nan, 1.0
    x[2] = -math.inf
    x[3] = math.nan
    x[3, 66666] = -math.inf
    rules, lists = make(4, 70000, 1)
    check(backend, x, rules, lists)
    pick = torch.empty(4, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(x, None, pick) and pick.tolist() == [9, 5, -1, -1]  # without rules or rows out
    # infinities, signed zeros: 0 and -0 are equal
    y = torch.tensor([[-1.0, -0.0, 0.0, -3.0], [1.0, math.inf, math.inf, 2.0]], device=DEV)
    pick = torch.empty(2, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(y, None, pick) and pick.tolist() == [1, 1]


def test_lists_and_masks_that_rows_share(backend):
    t, n = 3, 1000
    x = torch.randn((t, n), device=DEV)
    ids, b = [4, 999, 4, 17], [1.0, -100.0, -math.inf, 2.5]
    allowed = np.random.default_rng(2).random((1, n)) < 0.3
    rules = LogitRules(history=i32([5, 5, 999]), bias_ids=i32(ids), bias=torch.tensor(b, device=DEV), mask=torch.from_numpy(words_of(allowed)).to(DEV), **PENALTIES)
    check(backend, x, rules, {"history": [[5, 5, 999]] * t, "bias": [list(zip(ids, b))] * t, "allowed": np.repeat(allowed, t, 0)})
    rules.mask = rules.mask[0]
    check(backend, x, rules, {"history": [[5, 5, 999]] * t, "bias": [list(zip(ids, b))] * t, "allowed": np.repeat(allowed, t, 0)})


def test_nothing_left(backend):
    x = torch.randn((2, 5000), device=DEV)
    rules, lists = make(2, 5000, 3, mask=0.0)
    check(backend, x, rules, lists)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("shift", [0, 1])
def test_strides_alignments_and_results_in_place(backend, dtype, shift):
    t, n = 4, 9001
    room = torch.full((t * (n + 31 + shift) + shift,), 5.0, device=DEV, dtype=TYPES[dtype])
    view = room.as_strided((t, n), (n + 31 + shift, 1), shift)
    view.copy_(torch.randn((t, n), device=DEV))
    x = view.clone()
    rules, lists = make(t, n, 6, history=50, biases=10, mask=0.8, **PENALTIES)
    want, pick = plain(x, rules, lists)
    got = torch.empty(t, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(view, view, got, rules)
    assert torch.equal(view.cpu(), want) and got.tolist() == pick
    left = torch.ones_like(room, dtype=torch.bool)
    left.as_strided((t, n), (n + 31 + shift, 1), shift).fill_(False)
    assert (room[left] == 5.0).all()


def test_lists_that_do_not_fit_are_reported(backend):
    x = torch.randn((2, 100), device=DEV)
    for ptr in ([0, 3, 9], [0, -1, 2], [2, 1, 3]):
        rules = LogitRules(history=i32([1, 2, 3]), history_ptr=i32(ptr), **PENALTIES)
        out = torch.empty_like(x)
        assert backend.logits_dev(x, out, None, rules)
        torch.cuda.synchronize()
        with pytest.raises(ob.BackendError) as e:
            backend.check_status()
        assert e.value.code == -2 and "list" in str(e.value)
        backend.check_status()


def test_captured(backend):
    x = torch.randn((2, 40000), device=DEV)
    rules, lists = make(2, 40000, 8, history=50, mask=0.5, **PENALTIES)
    out, pick = torch.empty_like(x), torch.empty(2, dtype=torch.int32, device=DEV)
    assert backend.logits_dev(x, out, pick, rules)
    side = torch.cuda.Stream()
    backend.set_stream(side.cuda_stream)
    try:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            assert backend.logits_dev(x, out, pick, rules)
        for seed in (1, 2):
            x.copy_(torch.randn((2, 40000), device=DEV) * seed)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            want, w = plain(x, rules, lists)
            assert torch.equal(out.cpu(), want) and pick.tolist() == w
    finally:
        backend.set_stream(0)


def test_refusals(backend):
    x = torch.randn((2, 100), device=DEV)
    pick = torch.empty(2, dtype=torch.int32, device=DEV)
    for kw in (dict(repeat=0.0), dict(repeat=-1.0), dict(repeat=math.nan), dict(frequency=math.inf), dict(presence=math.nan)):
        with pytest.raises(ob.BackendError) as e:
            backend.logits_dev(x, x, pick, LogitRules(**kw))
        assert e.value.code == -2
    L = ob.lib()
    assert L.b2_logits_dev(backend._ctx, None, x.data_ptr(), 0, 2, 100, 100, 100, None, pick.data_ptr()) == -2
    assert L.b2_logits_dev(backend._ctx, x.data_ptr(), None, 0, 2, 100, 100, 100, None, None) == -2
    assert L.b2_logits_dev(backend._ctx, x.data_ptr(), x.data_ptr(), 5, 2, 100, 100, 100, None, None) == -2
    assert L.b2_logits_dev(backend._ctx, x.data_ptr(), x.data_ptr(), 0, 2, 100, 100, 99, None, None) == -2
    r = ob._lib.LogitRules(1.0, 0.0, 0.0, 4, 0)
    assert L.b2_logits_dev(backend._ctx, x.data_ptr(), x.data_ptr(), 0, 2, 100, 100, 100, C.byref(r), None) == -2  # a history without its list
    assert backend.logits_dev(x[:0], x[:0], pick[:0])
