"""What the operators between a decoder's products are measured on: the 8-bit cache, the attention that reads it, and the rules on logits.

``append``: new keys and values of several sequences go into a cache of 8-bit integers, a power of two as the scale of every block of 32 tokens,
head and kind; the blocks written are read back as the values that they stand for. ``attend``: queries over such a cache, one token a sequence
or a prompt, scores capped by a tanh, with a bias by distance, a window or a prefix that everybody sees. ``logits``: penalties for the tokens of
a history, biases and a grammar's mask on rows of logits, and the largest that is left.

``listed()`` holds the fixed cases, ``draw(rng)`` gives more of the same ranges. ``run`` computes the plain form, or, where ``own`` is
true, makes the calls that a program makes. Keys have channels of very different size, as decoders' keys do; all else follows from the seed.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
BLOCK = 32  # tokens of a block


def listed() -> list:
    return [
        # One decoding step of a serving batch: a token of each of 64 sequences, their blocks filled to various degrees.
        {"name": "append_b64_t1", "op": "append", "seqs": 64, "ctx": 2000, "rows": 1, "nkv": 8, "hd": 128, "dtype": "f32", "paged": True},
        # Chunks of several prompts together, ragged, heads of 64.
        {"name": "append_chunks", "op": "append", "seqs": 7, "ctx": 501, "rows": 700, "nkv": 8, "hd": 64, "dtype": "f16", "paged": True},
        # A long prompt of one sequence.
        {"name": "append_prompt8192", "op": "append", "seqs": 1, "ctx": 0, "rows": 8192, "nkv": 8, "hd": 128, "dtype": "bf16", "paged": False},
        # One token of one sequence, the context of the decode benchmark: latency.
        {"name": "attend_t1_ctx2048", "op": "attend", "seqs": 1, "ctx": 2048, "rows": 1, "nh": 32, "nkv": 8, "hd": 128, "dtype": "f32", "paged": False,
         "cap": 0.0, "window": 0, "bias": False, "prefix": 0},
        # One token of one sequence over a very long context.
        {"name": "attend_t1_ctx131071", "op": "attend", "seqs": 1, "ctx": 131071, "rows": 1, "nh": 32, "nkv": 8, "hd": 128, "dtype": "f32", "paged": False,
         "cap": 0.0, "window": 0, "bias": False, "prefix": 0},
        # A decoding step of a serving batch, contexts of every length up to 4096, scores capped.
        {"name": "attend_b64_ctx4096_cap", "op": "attend", "seqs": 64, "ctx": 4096, "rows": 1, "nh": 32, "nkv": 8, "hd": 128, "dtype": "bf16", "paged": True,
         "cap": 50.0, "window": 0, "bias": False, "prefix": 0},
        # Four drafted tokens of each of a few sequences, layers with a window, heads of 64.
        {"name": "attend_verify4_window", "op": "attend", "seqs": 9, "ctx": 5000, "rows": 4, "nh": 32, "nkv": 8, "hd": 64, "dtype": "f32", "paged": True,
         "cap": 0.0, "window": 1024, "bias": False, "prefix": 0},
        # Ragged prompts with a bias by distance, one KV head a query head.
        {"name": "attend_prompts_bias", "op": "attend", "seqs": 5, "ctx": 300, "rows": 600, "nh": 12, "nkv": 12, "hd": 128, "dtype": "f16", "paged": True,
         "cap": 0.0, "window": 0, "bias": True, "prefix": 0},
        # The second half of a prompt, the first 700 tokens of it seen by everybody: the largest case.
        {"name": "attend_prompt2048", "op": "attend", "seqs": 1, "ctx": 2048, "rows": 2048, "nh": 32, "nkv": 8, "hd": 128, "dtype": "bf16", "paged": False,
         "cap": 30.0, "window": 0, "bias": False, "prefix": 2700},
        # One token's choice: penalties for a conversation's tokens and a user's biases.
        {"name": "logits_t1", "op": "logits", "t": 1, "n": 128256, "history": 1500, "biases": 30, "mask": False, "dtype": "f32"},
        # The choices of a serving batch, each row under a grammar of its own.
        {"name": "logits_t64_mask", "op": "logits", "t": 64, "n": 128256, "history": 700, "biases": 0, "mask": True, "dtype": "f32"},
        # Many rows of a smaller vocabulary, everything at once.
        {"name": "logits_t256", "op": "logits", "t": 256, "n": 32064, "history": 4000, "biases": 300, "mask": True, "dtype": "bf16"},
    ]


def _log(rng, lo, hi) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    op = rng.choice(["append", "attend", "attend", "logits"])
    if op == "logits":
        t, n = _log(rng, 1, 256), _log(rng, 1000, 160000)
        while t * n > 8.2e6:
            t //= 2
        return {"op": op, "t": t, "n": n, "history": rng.choice([0, _log(rng, 1, 8000)]), "biases": rng.choice([0, _log(rng, 1, 300)]),
                "mask": rng.random() < 0.5, "dtype": rng.choice(["f32", "f32", "bf16", "f16"])}
    nkv, hd, dtype, paged = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 128]), rng.choice(["f32", "bf16", "f16"]), rng.random() < 0.6
    if op == "append":
        seqs, rows = _log(rng, 1, 64), rng.choice([1, _log(rng, 1, 8192)])
        while seqs * rows * nkv * hd > 8192 * 8 * 128:
            rows = rows // 2 + 1
            seqs = seqs // 2 + 1
        return {"op": op, "seqs": seqs, "ctx": rng.choice([0, _log(rng, 1, 4000)]), "rows": rows, "nkv": nkv, "hd": hd, "dtype": dtype, "paged": paged}
    group = rng.choice([1, 2, 4, 8])
    rows = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 2048)])
    seqs, ctx = _log(rng, 1, 64), rng.choice([0, _log(rng, 8, 100000)])
    while seqs * (ctx + rows) * nkv * hd > 64 * 4096 * 8 * 128 or seqs * rows * (ctx + rows) * nkv * group * hd > 2048 * 3000 * 32 * 128:
        if seqs > 1:
            seqs //= 2
        elif rows > ctx:
            rows //= 2
        else:
            ctx //= 2
    return {"op": op, "seqs": seqs, "ctx": ctx, "rows": rows, "nh": nkv * group, "nkv": nkv, "hd": hd, "dtype": dtype, "paged": paged,
            "cap": rng.choice([0.0, 0.0, 20.0, 50.0]), "window": rng.choice([0, 0, _log(rng, 16, 4096)]), "bias": rng.random() < 0.25,
            "prefix": rng.choice([0, 0, _log(rng, 1, 4096)])}


# ---- inputs ------------------------------------------------------------------------------------------------------------------------
def _ragged(case):
    """Positions where the sequences' rows begin, and how many rows each has (a case's own: its results have one shape)."""
    n, ctx, rows = case["seqs"], case["ctx"], case["rows"]
    rng = np.random.default_rng([n, ctx, rows])
    if n == 1:
        return [ctx], [rows]
    start = [int(v) for v in rng.integers(ctx // 4, ctx + 1, n)]
    if rows <= 8:
        return start, [rows] * n
    return start, [int(v) for v in rng.integers(rows // 4 + 1, rows + 1, n)]


class State:
    pass


def _layout(case, seed):
    """The sequences of a call: where their rows lie, and the blocks of the cache that they have."""
    rng = np.random.default_rng(seed)
    s = State()
    s.start, s.count = _ragged(case)
    s.length = [a + b for a, b in zip(s.start, s.count)]
    s.first = [0] + [int(v) for v in np.cumsum(s.count)]
    s.n_rows = s.first[-1]
    s.max_blocks = max(-(-n // BLOCK) for n in s.length)
    s.n_blocks = s.max_blocks * case["seqs"]
    ids = np.arange(s.n_blocks)
    if case["paged"]:
        rng.shuffle(ids)
    s.table = ids.reshape(case["seqs"], s.max_blocks)
    return s


def _gen(seed, *more):
    g = torch.Generator(device=DEV)
    g.manual_seed((seed * 1000003 + sum((i + 1) * 7919 * m for i, m in enumerate(more))) % (1 << 62))
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEV, generator=g)


def _keys_values(case, seed, seq, n, part):
    """Keys and values [n][nkv][hd] of a sequence: channels of different size, a few of them far larger; values smaller."""
    nkv, hd = case["nkv"], case["hd"]
    gain = torch.exp(0.4 * _randn(_gen(seed, 1), nkv, hd))
    gain = torch.where(torch.rand((nkv, hd), device=DEV, generator=_gen(seed, 2)) < 0.03, 6.0 * gain, gain)
    g = _gen(seed, 3, seq, part)
    k = _randn(g, n, nkv, hd) * gain
    v = _randn(g, n, nkv, hd) * 0.4
    return k.to(DTYPES[case["dtype"]]), v.to(DTYPES[case["dtype"]])


def _queries(case, s, seed):
    # scores of a standard deviation of about two, whatever the keys' channels
    q = _randn(_gen(seed, 4), s.n_rows, case["nh"], case["hd"]) * 1.2
    return q.to(DTYPES[case["dtype"]])


def _slopes(case):
    return torch.tensor([2.0 ** (-8.0 * (i + 1) / case["nh"]) for i in range(case["nh"])], device=DEV) if case["bias"] else None


def _scale(case):
    return float(np.float32(1.0 / math.sqrt(case["hd"])))


def _logit_inputs(case, seed):
    t, n = case["t"], case["n"]
    s = State()
    s.logits = (_randn(_gen(seed, 5), t, n) * 2.5).to(DTYPES[case["dtype"]])
    rng = np.random.default_rng(seed + 17)
    s.repeat, s.frequency, s.presence = 1.15, 0.2, 0.3
    if case["history"]:  # tokens repeat as words do
        counts = rng.integers(case["history"] // 2, case["history"] + 1, t)
        s.history_ptr = np.concatenate([[0], np.cumsum(counts)])
        s.history = np.minimum(np.exp(rng.uniform(0, math.log(n), int(s.history_ptr[-1]))), n - 1).astype(np.int64)
    else:
        s.history = None
    if case["biases"]:
        counts = rng.integers(0, case["biases"] + 1, t)
        s.bias_ptr = np.concatenate([[0], np.cumsum(counts)])
        s.bias_ids = np.concatenate([rng.choice(n, c, replace=False) for c in counts]).astype(np.int64)
        s.bias = rng.uniform(-6, 6, len(s.bias_ids)).astype(np.float32)
        if len(s.bias):
            s.bias[rng.random(len(s.bias)) < 0.1] = -100.0
    else:
        s.bias_ids = None
    if case["mask"]:  # a few tokens allowed in some rows, nearly all in the others
        share = torch.from_numpy(np.where(rng.random(t) < 0.5, 0.002, 0.9)).to(DEV)
        s.allowed = torch.rand((t, n), device=DEV, generator=_gen(seed, 6)) < share[:, None]
        s.allowed[:, 7 % n] = True
        pad = torch.zeros((t, -n % 32), dtype=torch.bool, device=DEV)
        bits = torch.cat([s.allowed, pad], 1).view(t, -1, 32).long() << torch.arange(32, device=DEV)
        words = bits.sum(-1)
        s.mask = torch.where(words >= 1 << 31, words - (1 << 32), words).int()
    else:
        s.allowed = None
    return s


# ---- plain forms -------------------------------------------------------------------------------------------------------------------
def _exponent(amax):
    """The smallest e with amax <= 127 * 2^e, at least -100."""
    m, e = torch.frexp(amax.double() / 127.0)
    e = torch.where(m == 0.5, e - 1, e)
    return torch.where(amax > 0, e, torch.full_like(e, -100)).clamp(min=-100)


def _plain_append(s, k, v):
    """Blocks [touched][2][nkv][32][hd] of integers: what was there before the new rows at the new scale, the new rows at it, what lies behind as it was."""
    new = torch.zeros((len(s.touched), BLOCK, 2) + tuple(k.shape[1:]), device=DEV)
    new[s.row_block, s.row_at, 0] = k.float()
    new[s.row_block, s.row_at, 1] = v.float()
    new = new.permute(0, 2, 3, 1, 4)  # [touched][2][nkv][32][hd]
    old, old_scale = s.cache[s.touched], s.scales[s.touched]
    e_new = _exponent(new.abs().amax(dim=(3, 4)))
    _, e_old = torch.frexp(old_scale)
    kept = (s.before > 0)[:, None, None] & (old_scale > 0)
    e = torch.where(kept, torch.maximum(e_new, e_old - 1), e_new)
    scale = torch.ldexp(torch.ones_like(old_scale), e)
    grown = torch.round(old.float() * torch.where(kept, old_scale / scale, torch.zeros_like(scale))[..., None, None])
    q = torch.round(new / scale[..., None, None])
    is_new = s.is_new[:, None, None, :, None]
    was = (torch.arange(BLOCK, device=DEV)[None, :] < s.before[:, None])[:, None, None, :, None]
    s.cache[s.touched] = torch.where(is_new, q, torch.where(was, grown, old.float())).to(torch.int8)
    s.scales[s.touched] = scale


def _plain_read(s):
    x = s.cache[s.read_block, :, :, s.read_at].float() * s.scales[s.read_block][..., None]  # [rows][2][nkv][hd]
    return x[:, 0].contiguous(), x[:, 1].contiguous()


def _quantize(x):
    """Integers and scales of whole blocks [blocks][32][nkv][hd]."""
    x = x.float()
    scale = torch.ldexp(torch.ones((), device=DEV), _exponent(x.abs().amax(dim=(1, 3))))  # [blocks][nkv]
    return torch.round(x / scale[:, None, :, None]).to(torch.int8), scale


def _fill_plain(s, case, seq, k, v):
    pad = -k.shape[0] % BLOCK
    blocks = torch.from_numpy(s.table[seq, : (k.shape[0] + pad) // BLOCK]).to(DEV)
    for i, x in enumerate((k, v)):
        x = torch.cat([x, torch.zeros((pad,) + tuple(x.shape[1:]), device=DEV, dtype=x.dtype)])
        q, scale = _quantize(x.view(-1, BLOCK, *x.shape[1:]))
        s.cache[blocks, i] = q.permute(0, 2, 1, 3)
        s.scales[blocks, i] = scale


def _plain_attend(s):
    case, out = s.case, torch.empty_like(s.q)
    nkv, hd = case["nkv"], case["hd"]
    G = case["nh"] // nkv
    for i in range(case["seqs"]):
        t, n = s.count[i], s.length[i]
        p = torch.arange(s.start[i], n, device=DEV)
        lo = max(0, s.start[i] - case["window"] + 1) // BLOCK if case["window"] else 0
        blocks = s.table_dev[i, lo : -(-n // BLOCK)]
        x = s.cache[blocks].float() * s.scales[blocks][..., None, None]  # [blocks][2][nkv][32][hd]
        k, v = x.permute(1, 2, 0, 3, 4).reshape(2, nkv, -1, hd)[:, :, : n - lo * BLOCK]
        j = torch.arange(lo * BLOCK, n, device=DEV)
        hidden = ~((j[None] <= p[:, None]) | (j[None] < case["prefix"]))
        if case["window"]:
            hidden |= p[:, None] - j[None] >= case["window"]
        q = s.q[s.first[i] : s.first[i + 1]].float().view(t, nkv, G, hd)
        y = torch.empty((t, nkv, G, hd), device=DEV)
        for h in range(nkv):
            sc = torch.matmul(q[:, h].reshape(t * G, hd), k[h].T).view(t, G, -1) * _scale(case)
            if case["cap"]:
                sc = case["cap"] * torch.tanh(sc / case["cap"])
            if s.slopes is not None:
                sc = sc + s.slopes[h * G : (h + 1) * G][None, :, None] * (j[None] - p[:, None])[:, None, :]
            sc = sc.masked_fill(hidden[:, None, :], -math.inf)
            w = torch.exp(sc - sc.amax(-1, keepdim=True))
            y[:, h] = (torch.matmul(w.view(t * G, -1), v[h]) / w.sum(-1).view(t * G, 1)).view(t, G, hd)
        out[s.first[i] : s.first[i + 1]] = y.view(t, nkv * G, hd).to(out.dtype)
    return out


def _plain_logits(s):
    case, x = s.case, s.logits.float()
    t, n = x.shape
    if s.history is not None:
        seen = torch.zeros((t, n), device=DEV).index_put_((s.history_row, s.history_dev), torch.ones((), device=DEV), accumulate=True)
        y = torch.where(x > 0, x / s.repeat_dev, x * s.repeat_dev) - (seen * s.frequency_dev + s.presence_dev)
        x = torch.where(seen > 0, y, x)
    if s.bias_ids is not None:
        b = torch.zeros((t, n), device=DEV).index_put_((s.bias_row, s.bias_ids_dev), s.bias_dev)
        x = x + b
    if s.allowed is not None:
        x = torch.where(s.allowed, x, torch.full((), -math.inf, device=DEV))
    out = x.to(s.logits.dtype)
    at = torch.where(out == out.amax(1, keepdim=True), torch.arange(n, device=DEV), n).amin(1)
    return out, at.int()


# ---- state and pass ------------------------------------------------------------------------------------------------------------------
_be = None


def _backend():
    global _be
    from oxinfer_b200 import Backend

    if _be is None:
        _be = Backend(0)
    _be.set_stream(torch.cuda.current_stream().cuda_stream)
    return _be


def _i32(v):
    return torch.from_numpy(np.asarray(v, dtype=np.int32)).to(DEV)


def _own_seqs(s, case, start, count):
    from oxinfer_b200.kv8 import Kv8Seqs

    first = np.concatenate([[0], np.cumsum(count)])
    return Kv8Seqs(start=_i32(start), rows=_i32(first), n_rows=int(first[-1]), max_rows=max(count), max_blocks=s.max_blocks,
                   table=_i32(s.table) if case["paged"] else None)


def prepare(case: dict, seed: int):
    if case["op"] == "logits":
        s = _logit_inputs(case, seed)
        s.case, t = case, case["t"]
        if own:
            from oxinfer_b200.sampling import LogitRules

            s.be, s.out, s.pick = _backend(), torch.empty_like(s.logits), torch.empty(t, dtype=torch.int32, device=DEV)
            rules = {}
            if s.history is not None:
                rules.update(repeat=s.repeat, frequency=s.frequency, presence=s.presence, history=_i32(s.history), history_ptr=_i32(s.history_ptr))
            if s.bias_ids is not None:
                rules.update(bias_ids=_i32(s.bias_ids), bias=torch.from_numpy(s.bias).to(DEV), bias_ptr=_i32(s.bias_ptr))
            if s.allowed is not None:
                rules.update(mask=s.mask)
            s.rules = LogitRules(**rules)
            return s
        s.repeat_dev, s.frequency_dev, s.presence_dev = (torch.tensor(v, device=DEV, dtype=torch.float32) for v in (s.repeat, s.frequency, s.presence))
        if s.history is not None:
            s.history_dev = torch.from_numpy(s.history).to(DEV)
            s.history_row = torch.repeat_interleave(torch.arange(t, device=DEV), torch.from_numpy(np.diff(s.history_ptr)).to(DEV))
        if s.bias_ids is not None:
            s.bias_ids_dev, s.bias_dev = torch.from_numpy(s.bias_ids).to(DEV), torch.from_numpy(s.bias).to(DEV)
            s.bias_row = torch.repeat_interleave(torch.arange(t, device=DEV), torch.from_numpy(np.diff(s.bias_ptr)).to(DEV))
        return s

    s = _layout(case, seed)
    s.case, nkv, hd, n = case, case["nkv"], case["hd"], case["seqs"]
    held = s.start if case["op"] == "append" else s.length  # tokens in the cache before the pass
    if own:
        s.be = _backend()
        s.cache = s.be.kv8(nkv, hd, s.n_blocks)
        assert s.cache is not None, s.be.last_declined
        for i in range(n):
            if held[i]:
                k, v = _keys_values(case, seed, i, held[i], 0)
                one = State()
                one.max_blocks, one.table = s.max_blocks, s.table[i : i + 1]
                assert s.cache.append(_own_seqs(one, {"paged": True}, [0], [held[i]]), k, v)
    else:
        s.cache = torch.zeros((s.n_blocks, 2, nkv, BLOCK, hd), dtype=torch.int8, device=DEV)
        s.scales = torch.zeros((s.n_blocks, 2, nkv), device=DEV)
        for i in range(n):
            if held[i]:
                _fill_plain(s, case, i, *_keys_values(case, seed, i, held[i], 0))
    if case["op"] == "append":
        kv = [_keys_values(case, seed, i, s.count[i], 1) for i in range(n)]
        s.k, s.v = torch.cat([x[0] for x in kv]), torch.cat([x[1] for x in kv])
        base = [a // BLOCK * BLOCK for a in s.start]
        span = [b - a for a, b in zip(base, s.length)]
        if own:
            s.seqs, s.back = _own_seqs(s, case, s.start, s.count), _own_seqs(s, case, base, span)
            s.k_back, s.v_back = (torch.empty((sum(span), nkv, hd), device=DEV) for _ in range(2))
        else:
            touched, before, is_new, row_block, row_at, read_block, read_at = [], [], [], [], [], [], []
            for i in range(n):
                for b in range(s.start[i] // BLOCK, -(-s.length[i] // BLOCK)):
                    lo, hi = max(s.start[i] - b * BLOCK, 0), min(s.length[i] - b * BLOCK, BLOCK)
                    row_block += [len(touched)] * (hi - lo)
                    row_at += list(range(lo, hi))
                    read_block += [s.table[i, b]] * hi
                    read_at += list(range(hi))
                    touched.append(s.table[i, b])
                    before.append(lo)
                    is_new.append([lo <= r < hi for r in range(BLOCK)])
            s.touched, s.before, s.is_new, s.row_block, s.row_at, s.read_block, s.read_at = (
                torch.from_numpy(np.asarray(x)).to(DEV) for x in (touched, before, is_new, row_block, row_at, read_block, read_at))
        return s
    s.q, s.slopes = _queries(case, s, seed), _slopes(case)
    if own:
        s.out, s.seqs = torch.empty_like(s.q), _own_seqs(s, case, s.start, s.count)
        s.prefix = _i32([case["prefix"]] * n) if case["prefix"] else None
    else:
        s.table_dev = torch.from_numpy(s.table).to(DEV)
    return s


def run(s):
    case = s.case
    if case["op"] == "logits":
        if not own:
            return _plain_logits(s)
        done = s.be.logits_dev(s.logits, s.out, s.pick, s.rules)
        assert done, s.be.last_declined
        return s.out, s.pick
    if case["op"] == "append":
        if not own:
            _plain_append(s, s.k, s.v)
            return _plain_read(s)
        done = s.cache.append(s.seqs, s.k, s.v) and s.cache.read(s.back, s.k_back, s.v_back)
        assert done, s.be.last_declined
        return s.k_back, s.v_back
    if not own:
        return _plain_attend(s)
    done = s.cache.attend(s.seqs, s.q, s.out, scale=_scale(case), cap=case["cap"], window=case["window"], slopes=s.slopes, prefix=s.prefix)
    assert done, s.be.last_declined
    return s.out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------------------------
def _visible(case, start, count):
    """(Query, key) pairs that are seen, and the keys that some query sees."""
    n = start + count
    p = np.arange(start, n, dtype=np.int64)
    last = np.maximum(p + 1, min(case["prefix"], n))
    first = np.maximum(p + 1 - case["window"], 0) if case["window"] else np.zeros_like(p)
    pairs = int(np.sum(last - first))
    return pairs, int(last.max() - first.min())


def work(case: dict) -> dict:
    if case["op"] == "logits":
        t, n = case["t"], case["n"]
        touched = t * (0.75 * case["history"] * 4 + 0.5 * case["biases"] * 8)
        return {"bytes": t * n * 2 * SIZE[case["dtype"]] + touched + (t * n / 8 if case["mask"] else 0) + 4 * t, "flops": 2.0 * t * n}
    s = _layout(case, 0)
    row = case["nkv"] * case["hd"] * 2  # keys and values of a token
    if case["op"] == "append":
        back = sum(n - a // BLOCK * BLOCK for a, n in zip(s.start, s.length))  # rows of the blocks written
        return {"bytes": s.n_rows * row * (SIZE[case["dtype"]] + 1) + back * row * (1 + 4), "flops": 2.0 * s.n_rows * row}
    seen = [_visible(case, a, c) for a, c in zip(s.start, s.count)]
    heads = case["nh"] * case["hd"]
    return {"bytes": sum(k for _, k in seen) * (row + 8 * case["nkv"] / BLOCK) + 2 * s.n_rows * heads * SIZE[case["dtype"]],
            "flops": 4.0 * heads * sum(p for p, _ in seen)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------------
def _exact_block(old, old_scale, new):
    """A block's rows after `new` rows behind `old` ones (integers at `old_scale`), one head and kind: integers and their scale."""
    top = np.abs(new).max(axis=(0, 2))  # a head
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(top / 127.0))
    e = np.maximum(np.where(top <= 127.0 * 2.0 ** (e - 1), e - 1, np.where(top > 127.0 * 2.0 ** e, e + 1, e)), -100)
    scale = 2.0 ** e
    if len(old):
        scale = np.maximum(scale, old_scale)
        old = np.rint(old * (old_scale / scale)[None, :, None])
    return np.concatenate([old, np.rint(new / scale[None, :, None])]), scale


def _exact_rows(x):
    """Values that rows [n][nkv][hd], written at once from a block's beginning on, stand for."""
    x = x.double().cpu().numpy()
    out = []
    for a in range(0, len(x), BLOCK):
        q, scale = _exact_block(x[:0], None, x[a : a + BLOCK])
        out.append(q * scale[None, :, None])
    return np.concatenate(out)


def _exact_append(case, seed):
    s = _layout(case, seed)
    backs = ([], [])
    for i in range(case["seqs"]):
        before = _keys_values(case, seed, i, s.start[i], 0) if s.start[i] else None
        added = _keys_values(case, seed, i, s.count[i], 1)
        for kind in range(2):
            new = added[kind].double().cpu().numpy()
            lead, at = s.start[i] % BLOCK, 0
            if lead:
                had = before[kind][s.start[i] - lead :].double().cpu().numpy()
                q0, sc0 = _exact_block(had[:0], None, had)
                at = min(BLOCK - lead, len(new))
                q, sc = _exact_block(q0, sc0, new[:at])
                backs[kind].append(q * sc[None, :, None])
            if at < len(new):
                backs[kind].append(_exact_rows(torch.from_numpy(new[at:])))
    return tuple(torch.from_numpy(np.concatenate(b)) for b in backs)


def _exact_attend(case, seed):
    s = _layout(case, seed)
    q = _queries(case, s, seed).double()
    slopes = _slopes(case)
    G, outs = case["nh"] // case["nkv"], []
    for i in range(case["seqs"]):
        k, v = (torch.from_numpy(_exact_rows(x)).to(DEV) for x in _keys_values(case, seed, i, s.length[i], 0))
        pos = torch.arange(s.length[i], device=DEV)
        qi = q[s.first[i] : s.first[i + 1]]
        y = torch.empty_like(qi)
        for a in range(0, s.count[i], 512):
            p = pos[s.start[i] + a : s.start[i] + min(a + 512, s.count[i])]
            see = (pos[None] <= p[:, None]) | (pos[None] < case["prefix"])
            if case["window"]:
                see &= p[:, None] - pos[None] < case["window"]
            for h in range(case["nh"]):
                sc = qi[a : a + 512, h] @ k[:, h // G].T * _scale(case)
                if case["cap"]:
                    sc = case["cap"] * torch.tanh(sc / case["cap"])
                if slopes is not None:
                    sc = sc + slopes[h].double() * (pos[None] - p[:, None])
                y[a : a + 512, h] = torch.softmax(torch.where(see, sc, -math.inf), -1) @ v[:, h // G]
        outs.append(y)
    return torch.cat(outs)


def _exact_logits(case, seed):
    s = _logit_inputs(case, seed)
    x = s.logits.double().cpu().numpy()
    repeat, frequency, presence = (float(np.float32(v)) for v in (s.repeat, s.frequency, s.presence))
    for i in range(case["t"]):
        if s.history is not None:
            ids, counts = np.unique(s.history[s.history_ptr[i] : s.history_ptr[i + 1]], return_counts=True)
            was = x[i, ids]
            x[i, ids] = np.where(was > 0, was / repeat, was * repeat) - (frequency * counts + presence)
        if s.bias_ids is not None:
            part = slice(s.bias_ptr[i], s.bias_ptr[i + 1])
            x[i, s.bias_ids[part]] += s.bias[part].astype(np.float64)
    if s.allowed is not None:
        x[~s.allowed.cpu().numpy()] = -np.inf
    # the choice is among the values as they are stored
    stored = torch.from_numpy(x).to(DTYPES[case["dtype"]]).float().numpy()
    return torch.from_numpy(x), torch.from_numpy(stored.argmax(1).astype(np.int32))


def exact(case: dict, seed: int):
    return {"append": _exact_append, "attend": _exact_attend, "logits": _exact_logits}[case["op"]](case, seed)
