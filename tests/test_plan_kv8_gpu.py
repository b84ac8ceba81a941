"""Plans with 8-bit caches (B2_KV_I8): the ops on them against the definition in 64 bits, rows in and out, whole decoders, and generation under rules."""
import numpy as np
import pytest

import oxinfer_b200 as ob
from oracle import oracle as O
from oxinfer_b200 import decode as D
from oxinfer_b200 import synth
from oxinfer_b200.sampling import GenerateRules

from test_kv8_gpu import Model

pytestmark = pytest.mark.gpu

SMALL = dict(n_layers=2, h=256, nh=4, nkv=2, hd=64, inter=512, vocab=1024)


def attention_graph(nh, nkv, hd, interleaved, window, norms):
    """A graph of rotation and attention alone: a step's input is q | k | v, its hidden state the heads' outputs."""
    g = D.Graph()
    qkv, qo, att = g.buf((nh + 2 * nkv) * hd), g.buf(nh * hd), g.buf(nh * hd)
    g.input, g.n_input, g.hidden, g.n_hidden, g.rope_halves = qkv, (nh + 2 * nkv) * hd, att, nh * hd, [hd // 2]
    g.kv.append((nkv, hd))
    g.qk_rope(qkv, qo, 0, nh, nkv, hd, hd // 2, nh * hd, (nh + nkv) * hd, interleaved, 1e-5, q_norm=norms, k_norm=norms)
    g.attend(qo, att, 0, nh, nkv, hd, float(1 / np.sqrt(hd)), window)
    return g


def rotate(x, cs, interleaved):
    """x [t][heads][hd] f32, cs [t][hd]; products and sums rounded one by one, as the kernels do."""
    half = x.shape[-1] // 2
    c, s = cs[:, None, :half], cs[:, None, half:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :half], x[..., half:])
    y = np.empty_like(x)
    p, q = a * c - b * s, b * c + a * s
    if interleaved:
        y[..., 0::2], y[..., 1::2] = p, q
    else:
        y[..., :half], y[..., half:] = p, q
    return y


def attend64(q, k, v, pos, window):
    """q [t][nh][hd] at positions pos ..; and the bound of the attention's own test: 2^-18.5 of the magnitudes in a score and 2^-19 of the largest value."""
    t, nh, hd = q.shape
    G = nh // k.shape[1]
    y, tol = np.zeros((t, nh, hd)), np.zeros((t, nh, 1))
    for i in range(t):
        first = max(0, pos + i + 1 - window) if window else 0
        for h in range(nh):
            kk, vv, qq = k[first:pos + i + 1, h // G], v[first:pos + i + 1, h // G], q[i, h].astype(np.float64)
            sc = kk @ qq / np.sqrt(hd)
            w = np.exp(sc - sc.max())
            y[i, h] = w @ vv / w.sum()
            tol[i, h] = np.abs(vv).max() * (2.0 ** -18.5 * (np.abs(kk) @ np.abs(qq)).max() / np.sqrt(hd) + 2.0 ** -19)
    return y.reshape(t, -1), np.broadcast_to(tol, (t, nh, hd)).reshape(t, -1)


def split(x, nh, nkv, hd):
    x = x.reshape(len(x), -1, hd)
    return x[:, :nh], x[:, nh:nh + nkv], x[:, nh + nkv:]


@pytest.mark.parametrize("kind", ["one", "multi", "prefill"])
@pytest.mark.parametrize("nh,nkv,hd,interleaved,window", [(4, 2, 64, True, 0), (8, 1, 128, False, 0), (6, 2, 128, True, 40), (3, 3, 64, False, 7)])
def test_steps_append_and_attend(backend, kind, nh, nkv, hd, interleaved, window):
    max_len = 200
    g = attention_graph(nh, nkv, hd, interleaved, window, None)
    plan = {"one": lambda: D.decode_plan(backend, g, max_len, kv_i8=True), "multi": lambda: D.decode_plan_multi(backend, g, max_len, 4, kv_i8=True),
            "prefill": lambda: D.decode_plan_prefill(backend, g, max_len, 90, kv_i8=True)}[kind]()
    assert plan is not None, backend.last_declined
    rng = np.random.default_rng(7)
    model, inv, pos = Model(nkv, hd, -(-max_len // 32)), D.rope_inv_freq(hd, 10000.0), 0
    steps = {"one": [1] * 70, "multi": [1, 4, 3, 2, 4, 4, 4, 4, 4, 1, 4, 4], "prefill": [1, 5, 31, 90, 2, 71]}[kind]
    for n, t in enumerate(steps):
        if n == 8:
            pos -= 3  # drafted tokens that were not accepted
        x = (rng.standard_normal((t, g.n_input)) * np.exp(rng.normal(0, 1, (t, 1)))).astype(np.float32)
        cs = np.stack([D.rope_table(pos + i, inv) for i in range(t)])
        got = plan.step(pos, x[0], cs[0], want_logits=False)[0][None] if kind == "one" else plan.step_multi(pos, x, cs, want_logits=False)[0]
        q, k, v = split(x, nh, nkv, hd)
        q, k = rotate(q, cs, interleaved), rotate(k, cs, interleaved)
        model.append(pos, k, v)
        kv = model.values(pos + t)
        for a, b in zip(plan.kv_read(0, 0, pos + t), kv):
            assert np.array_equal(a, b), (n, pos)
        want, tol = attend64(q, *kv, pos, window)
        if kind == "prefill" and t * (nh // nkv) >= 64:
            # many rows of a prefill step are multiplied as f16: each query value is off by 2^-11 of itself, so a score by 2^-11 of the magnitudes in it and a
            # probability by twice that (and its own rounding, 2^-11), where the bound above has 2^-18.5 of them: 2^8.5 as much, and 2^-10 of the largest value
            tol = tol * 2.0 ** 8.5 + 2.0 ** -10 * np.abs(kv[1]).max()
        assert (np.abs(got - want) <= tol).all(), (n, pos, np.abs(got - want).max())
        pos += t
    plan.close()


def test_per_head_norms_run_ahead_of_the_rounding(backend):
    nh, nkv, hd = 4, 2, 64
    norms = np.linspace(0.5, 1.5, hd).astype(np.float32)
    g = attention_graph(nh, nkv, hd, True, 0, norms)
    f32, i8 = D.decode_plan(backend, g, 64), D.decode_plan(backend, g, 64, kv_i8=True)
    rng = np.random.default_rng(9)
    cs = D.rope_table(5, D.rope_inv_freq(hd, 10000.0))
    x = rng.standard_normal(g.n_input).astype(np.float32)
    f32.step(5, x, cs, want_logits=False), i8.step(5, x, cs, want_logits=False)
    model = Model(nkv, hd, 1)
    k, v = f32.kv_read(0, 5, 1)
    model.append(0, k, v)
    for a, b in zip(i8.kv_read(0, 5, 1), model.values(1)):
        assert np.array_equal(a, b)
    f32.close(), i8.close()


def test_rows_in_and_out(backend):
    """kv_write keeps a block's other rows, brought to its scale; what kv_read gives goes back in unchanged."""
    nh, nkv, hd, max_len = 2, 2, 128, 700
    plan = D.decode_plan(backend, attention_graph(nh, nkv, hd, True, 0, None), max_len, kv_i8=True)
    other = D.decode_plan(backend, attention_graph(nh, nkv, hd, True, 0, None), max_len, kv_i8=True)
    rng = np.random.default_rng(10)
    held = np.zeros((2, max_len, nkv, hd))
    top = np.zeros((2, -(-max_len // 32), nkv))  # of each block, of all that was ever written into it since it was last written whole
    for pos, n, size in [(0, 600, 1.0), (40, 1, 0.01), (100, 3, 5.0), (31, 2, 20.0), (64, 32, 0.1), (1, 599, 1.0), (257, 443, 2.0), (0, 0, 1.0)]:
        kv = (rng.standard_normal((2, n, nkv, hd)) * size).astype(np.float32)
        plan.kv_write(0, pos, *kv) if n else None
        held[:, pos:pos + n] = kv
        got = np.stack(plan.kv_read(0, 0, max_len)).astype(np.float64)
        for b in range(-(-max_len // 32)):
            lo, hi = max(pos, 32 * b), min(pos + n, 32 * b + 32, max_len)
            if lo >= hi:
                continue
            new = np.abs(held[:, lo:hi]).max(axis=(1, 3))
            top[:, b] = new if hi - lo == 32 else np.maximum(top[:, b], new)
        step = 2.0 ** np.ceil(np.log2(np.maximum(top, 1e-30) / 127.0)).repeat(32, 1)[:, :max_len, :, None]
        # a row is rounded by half a step when it is written, and by half of the block's step at most in all when that has grown (1/2 + 1/4 + ..: less than one)
        assert (np.abs(got - held) <= step).all(), (pos, n)
    again = np.stack(plan.kv_read(0, 0, max_len))
    other.kv_write(0, 0, *again)
    assert np.array_equal(np.stack(other.kv_read(0, 0, max_len)), again)
    again[0, 5, 1, 3], again[1, 699, 0, 0] = np.nan, np.inf
    other.kv_write(0, 0, *again)
    back = np.stack(other.kv_read(0, 0, max_len))
    again[0, 5, 1], again[1, 699, 0] = np.nan, np.nan
    assert np.array_equal(back, again, equal_nan=True)
    plan.close(), other.close()


def llama(backend, cfg, seed):
    layers, final_norm, head, embed, shapes = synth.llama_weights(seed=seed, **cfg)
    dev = []
    for L in layers:
        d = {name: backend.upload(L[name], n_out, n_in) for name, (n_out, n_in) in shapes.items()}
        d["ln_pre"], d["ln_post"] = L["ln_pre"], L["ln_post"]
        dev.append(d)
    lc = D.LlamaConfig(eps=1e-5, **cfg)
    dhead = backend.upload(head, cfg["vocab"], cfg["h"])
    demb = backend.upload(embed, cfg["vocab"], cfg["h"])
    return lc, dev, final_norm, dhead, demb


def rows(pos, t, inv):
    return np.stack([O.rope_table(pos + i, inv) for i in range(t)])


def test_a_prompt_its_caches_and_generation(backend):
    """A prompt through a prefill plan, its rows into a decode plan, tokens generated on the device: the tokens of steps with the choice made here."""
    lc, dev, norm, head, emb = llama(backend, SMALL, 31)
    pre = D.decode_plan_prefill(backend, D.llama_graph(lc, dev, norm, head, prefill=True), 300, 128, kv_i8=True)
    g = D.llama_graph(lc, dev, norm, head)
    plan, f32 = D.decode_plan(backend, g, 300, kv_i8=True), D.decode_plan(backend, g, 300)
    inv = O.rope_inv_freq(SMALL["hd"], lc.rope_theta)
    rng = np.random.default_rng(12)
    table = backend.dequantize_rows(emb)
    prompt = rng.integers(0, SMALL["vocab"], 128)
    hid, _ = pre.step_multi(0, table[prompt], rows(0, 128, inv))
    for li in range(SMALL["n_layers"]):
        k, v = pre.kv_read(li, 0, 128)
        plan.kv_write(li, 0, k, v), f32.kv_write(li, 0, k, v)
        assert np.array_equal(np.stack(plan.kv_read(li, 0, 128)), np.stack((k, v)))

    def by_hand(p, n, choose):
        tok, out = 7, []
        for i in range(n):
            _, logits = p.step(128 + i, table[tok], O.rope_table(128 + i, inv))
            tok = choose(logits, out)
            out.append(tok)
        return out

    want = by_hand(plan, 60, lambda l, _: int(l.argmax()))
    cs = rows(128, 100, inv)
    assert plan.generate(emb, 7, 128, 60, cs[:60])[0].tolist() == want

    def ruled(l, done, repeat, frequency, presence, first, bias, allowed):
        f = np.float32
        l = l.copy()
        for i, c in zip(*np.unique(first + done, return_counts=True)) if first + done else []:
            l[i] = (l[i] / f(repeat) if l[i] > 0 else l[i] * f(repeat)) - (f(c) * f(frequency) + f(presence))
        for i, b in bias.items():
            l[i] = l[i] + f(b)
        if allowed is not None:
            l[~allowed] = -np.inf
        return int(l.argmax())

    allowed = rng.random(SMALL["vocab"]) < 0.5
    words = np.packbits(allowed, bitorder="little").view(np.uint32)
    first = [int(v) for v in prompt]
    cases = [(dict(repeat=1.4), dict(first=first), 40), (dict(repeat=1.1, frequency=0.5, presence=0.2, prompt=prompt), dict(first=first), 40),
             (dict(bias_ids=[want[0], 3, 3], bias=[-50.0, 1.0, 2.5]), dict(bias={want[0]: -50.0, 3: 2.5}), 30), (dict(mask=words), dict(allowed=allowed), 30),
             (dict(frequency=0.3, prompt=prompt[:5], mask=words, bias_ids=[9], bias=[4.0]), dict(first=first[:5], bias={9: 4.0}, allowed=allowed), 60),
             (dict(), dict(), 30), (dict(repeat=1.4, prompt=prompt), dict(first=first), 100)]
    for rules, model, n in cases:
        if "prompt" not in rules:
            model.pop("first", None)
        m = dict(repeat=rules.get("repeat", 1.0), frequency=rules.get("frequency", 0.0), presence=rules.get("presence", 0.0), first=[], bias={}, allowed=None)
        m.update(model)
        tokens = by_hand(plan, n, lambda l, done: ruled(l, done, **m))
        assert plan.generate(emb, 7, 128, n, cs[:n], rules=GenerateRules(**rules))[0].tolist() == tokens, rules
        assert f32.generate(emb, 7, 128, n, cs[:n], rules=GenerateRules(**rules))[0].tolist() == by_hand(f32, n, lambda l, done: ruled(l, done, **m)), rules
    assert plan.generate(emb, 7, 128, 60, cs[:60])[0].tolist() == want  # and without rules again
    other = backend.upload(synth.make("q8_0", SMALL["vocab"], SMALL["h"], 5), SMALL["vocab"], SMALL["h"])  # another embedding, both ways
    a = plan.generate(other, 7, 128, 20, cs[:20], rules=GenerateRules())[0].tolist()
    assert plan.generate(other, 7, 128, 20, cs[:20])[0].tolist() == a
    assert plan.generate(emb, 7, 128, 60, cs[:60])[0].tolist() == want
    with pytest.raises(ob.BackendError):
        backend._check(backend._L.b2_free_weight(backend._ctx, emb.handle))
    for p in (pre, plan, f32):
        p.close()


def test_steps_of_several_tokens_are_the_same_from_run_to_run(backend):
    lc, dev, norm, head, emb = llama(backend, SMALL, 33)
    g = D.llama_graph(lc, dev, norm, head)
    inv = O.rope_inv_freq(SMALL["hd"], lc.rope_theta)
    x = np.random.default_rng(13).standard_normal((40, SMALL["h"])).astype(np.float32)
    runs = []
    for _ in range(2):
        many = D.decode_plan_multi(backend, g, 300, 4, kv_i8=True)
        runs.append(np.concatenate([np.concatenate(many.step_multi(4 * i, x[4 * i:4 * i + 4], rows(4 * i, 4, inv)), 1) for i in range(10)]))
        many.close()
    assert np.isfinite(runs[0]).all() and np.array_equal(*runs)


def test_refusals(backend):
    g = attention_graph(4, 2, 96, True, 0, None)
    assert D.decode_plan(backend, g, 64, kv_i8=True) is None and "head dimension" in backend.last_declined
    lc, dev, norm, head, emb = llama(backend, SMALL, 34)
    plan = D.decode_plan(backend, D.llama_graph(lc, dev, norm, head), 64, kv_i8=True)
    inv = O.rope_inv_freq(SMALL["hd"], lc.rope_theta)
    cs = rows(0, 4, inv)
    for kw in (dict(repeat=0.0), dict(repeat=np.nan), dict(presence=np.inf), dict(mask=np.zeros(32, np.uint32))):
        with pytest.raises(ob.BackendError) as e:
            plan.generate(emb, 1, 0, 4, cs, rules=GenerateRules(**kw))
        assert e.value.code == -2
    with pytest.raises(ob.BackendError):
        plan.step(64, np.zeros(SMALL["h"], np.float32), cs[0])
    assert len(plan.generate(emb, 1, 0, 4, cs, rules=GenerateRules())[0]) == 4
    plan.close()
