"""Calls of the 8-bit cache and of rules on logits that their documentation allows: strides, alignments, results over inputs, sizes of one and of none."""
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
