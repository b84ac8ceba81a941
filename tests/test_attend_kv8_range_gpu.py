"""Attention over the 8-bit cache where queries, values and probabilities are as far apart as their types allow."""
import math

import pytest
import torch

from oxinfer_b200.kv8 import Kv8Seqs

from test_attend_kv8_gpu import DEV, Setting, i32

pytestmark = pytest.mark.gpu


def test_a_dominant_key_ahead_of_a_long_flat_tail(backend):
    """131072 keys of 2^-26 of the first one's probability each are 2^-9 of the result together. 80 sequences of 64 rows share the keys, so a CTA has all of them."""
    n, seqs, t, hd = 131072, 80, 64, 64
    g = torch.Generator(device=DEV)
    g.manual_seed(31)
    cache = backend.kv8(1, hd, n // 32)
    k = torch.zeros((n, 1, hd), device=DEV)
    k[0, 0, 0] = 144.0  # (72 * 2 in the cache)
    v = 0.5 + 0.5 * torch.rand((n, 1, hd), device=DEV, generator=g)
    v[0] = 0.0
    assert cache.append(Kv8Seqs(start=i32([0]), max_rows=n, max_blocks=n // 32), k, v) and cache.read(Kv8Seqs(start=i32([0]), max_rows=n, max_blocks=n // 32), k, v)
    table = torch.arange(n // 32, dtype=torch.int32, device=DEV).expand(seqs, -1).contiguous()
    q = torch.zeros((seqs * t, 1, hd), dtype=torch.bfloat16, device=DEV)
    q[:, 0, 0] = 1.0
    out = torch.empty_like(q)
    assert cache.attend(Kv8Seqs(start=i32([n - t] * seqs), max_rows=t, max_blocks=n // 32, table=table), q, out, scale=0.125)
    w = torch.ones(n, dtype=torch.float64, device=DEV)
    w[0] = math.exp(18.0)
    y = (torch.cumsum(w[:, None] * v[:, 0].double(), 0) / torch.cumsum(w, 0)[:, None])[n - t:]
    # a probability's f16 rounding is at most 2^-11 of it (2^-25 of what the row's largest is at least 2^7 of, for the smallest), the scores' 2^-18.5 of 18, half a step of the result
    tol = (2.0 ** -11 + 18 * 2.0 ** -18.5 + torch.finfo(torch.bfloat16).eps / 2) * y + n * 2.0 ** -32
    assert ((out.view(seqs, t, hd).double() - y).abs() <= tol).all(), ((out.view(seqs, t, hd).double() - y).abs() / y).max()


@pytest.mark.parametrize("dtype,count", [("f32", 1), ("f32", 70), ("bf16", 1), ("bf16", 20), ("bf16", 140)])
def test_queries_up_to_the_largest(backend, dtype, count):
    for hd in (64, 128):
        s = Setting(backend, [300], [count], 4, 2, hd, dtype, seed=32, spread=1e-10)
        s.q = (s.q.float().clamp(-3.0, 3.0) * 1.1e38).to(s.dtype)
        s.q[0, 0, 5] = -3.3e38
        s.scale = 1e-28
        out = s.check()
        assert float((out[:, 0] - out[:, 1]).abs().max()) > 0.05


@pytest.mark.parametrize("dtype,counts,lengths", [("f32", [1, 3], [90, 200]), ("f32", [40, 70], [90, 200]), ("f32", [1], [40000]), ("bf16", [1, 2], [90, 200]), ("bf16", [9, 20], [90, 200]),
                                                  ("bf16", [64, 190], [90, 200]), ("bf16", [64], [9000])])
def test_values_up_to_the_largest(backend, dtype, counts, lengths):
    """Finite values give finite results: sums of probabilities times values stay below the largest f32 on the way."""
    for hd in (64, 128):
        s = Setting(backend, lengths, counts, 4, 2, hd, dtype, seed=33)
        n = sum(lengths)
        g = torch.Generator(device=DEV)
        g.manual_seed(34)
        v = torch.randn((n, 2, hd), device=DEV, generator=g).clamp(-1.0, 1.0) * 3e38
        every = Kv8Seqs(start=i32([0] * len(lengths)), rows=i32(s.first_of), n_rows=n, max_rows=max(lengths), max_blocks=s.max_blocks, table=s.table)
        k = s.k.clone()
        assert s.cache.append(every, k, v) and s.cache.read(every, s.k, s.v)
        assert torch.isfinite(s.check()).all() and torch.isfinite(s.check(cap=3.0, window=50)).all()


class Apart:
    """One sequence whose values are `size` [n] large, and the formula's results with a bound that goes by the largest value in a row's own sight."""

    def __init__(self, backend, size, t, nh, nkv, hd, seed, poison=()):
        n = size.numel()
        self.s = s = Setting(backend, [n], [t], nh, nkv, hd, "bf16", seed=seed)
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        v = torch.randn((n, nkv, hd), device=DEV, generator=g) * size[:, None, None].float()
        for pos, head in poison:
            v[pos, head, 3] = math.nan
        every = Kv8Seqs(start=i32([0]), max_rows=n, max_blocks=s.max_blocks, table=s.table)
        k = s.k.clone()
        assert s.cache.append(every, k, v) and s.cache.read(every, s.k, s.v)
        self.n, self.t = n, t

    def check(self, **kw):
        s, n, t = self.s, self.n, self.t
        y, _ = s.want(**kw)
        out = torch.full_like(s.q, 9.0)
        pre = i32(kw["prefix"]) if kw.get("prefix") is not None else None
        assert s.cache.attend(s.seqs, s.q, out, scale=s.scale, cap=kw.get("cap", 0.0), window=kw.get("window", 0), slopes=kw.get("slopes"), prefix=pre)
        torch.cuda.synchronize()
        s.be.check_status()
        j, p = torch.arange(n, device=DEV), torch.arange(n - t, n, device=DEV)
        see = j[None] <= p[:, None]
        if pre is not None:
            see |= j[None] < pre[0]
        if kw.get("window"):
            see &= p[:, None] - j[None] < kw["window"]
        top = (see[:, :, None] * s.v.nan_to_num(0.0).abs().amax(-1).double()[None]).amax(1)  # [t][nkv]: the largest value that a row sees
        top = top.repeat_interleave(s.nh // s.nkv, 1)[:, :, None]
        # 2^-11 of a probability, 2^-13 for the scores' rounding (2^-18.5 of magnitudes of up to 45), half a step of the result
        tol = top * (2.0 ** -11 + 2.0 ** -13) + torch.finfo(torch.bfloat16).eps / 2 * y.abs().nan_to_num(0.0)
        got = out.double()
        assert torch.equal(torch.isnan(got), torch.isnan(y))
        err = ((got - y).abs() - tol).nan_to_num(0.0)
        assert (err <= 0).all(), ((got - y).abs() / top.clamp(min=1e-300)).nan_to_num(0.0).max()
        return out


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("nh,nkv", [(2, 2), (8, 2), (6, 2)])
def test_large_values_reach_no_row_that_does_not_see_them(backend, nh, nkv, hd):
    """Values 2^31 to 2^45 apart: behind the rows that see the small ones, within one tile of keys, and in front of the window."""
    n = 400
    at = torch.arange(n, device=DEV)
    for size in (2.0 ** torch.where(at < 200, -45.0, 0.0), 2.0 ** torch.where(at < 200, 0.0, -45.0), 2.0 ** torch.where(at // 32 % 3 == 2, 1.0, torch.where(at // 32 % 3 == 1, -30.0, -31.0))):
        a = Apart(backend, size, 350, nh, nkv, hd, seed=35)
        a.check()
        a.check(window=20)
        a.check(cap=4.0, window=70, prefix=[90])
        a.check(slopes=torch.tensor([-0.05 * (i + 1) for i in range(nh)], device=DEV), prefix=[150])


def test_large_values_with_shares_and_what_is_not_finite(backend):
    at = torch.arange(5000, device=DEV)
    for size in (2.0 ** torch.where(at < 4960, -50.0, 3.0), 2.0 ** torch.where(at < 100, 3.0, -50.0), 2.0 ** torch.where(at % 1000 < 500, -40.0, 0.0)):
        a = Apart(backend, size, 80, 4, 2, 128, seed=36)
        a.check()
        a.check(window=30)
        a.check(window=600, cap=5.0)
        a = Apart(backend, size, 80, 4, 2, 64, seed=37, poison=[(4955, 1), (4500, 0)])
        out = a.check(window=50)
        assert torch.isnan(out[35:, 2:]).all() and not torch.isnan(out[:35]).any() and not torch.isnan(out[:, :2]).any()
    # the smallest scale there is, with values and without
    size = torch.where(at < 4960, 0.0, 1.0).double()
    size[4800:4900] = 2.0 ** -96
    Apart(backend, size, 300, 2, 1, 64, seed=38).check(window=130)
