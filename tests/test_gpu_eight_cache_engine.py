"""The engine over the cache held in 8 bits (half_kv = HE_KV_EIGHT), and its log probabilities (he_score, he_logprobs)."""
import ctypes
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import cache_lib as cl
import oracle_lib as ol
from paths import REPO, package
from plans import plan_of
from tiny import sharp_checkpoint

pytestmark = pytest.mark.gpu

FIELDS = dict(dim=64, hidden_dim=128, n_layers=2, n_heads=4, n_kv_heads=2, head_size=16, vocab_size=320, seq_len=300,
              shared_classifier=1)
FORMS = {
    "llama": FIELDS,
    "qwen int6": dict(FIELDS, n_heads=2, n_kv_heads=1, head_size=32, six=1, qkv_bias=1, shared_classifier=0),
    "qwen3": dict(FIELDS, qk_norm=1),
    "gpt2": dict(FIELDS, n_kv_heads=4, arch=1, relaxed=0),
    "neox": dict(FIELDS, n_kv_heads=4, arch=2, rotary=8, parallel_residual=1),
    "wide heads": dict(FIELDS, dim=256, n_heads=2, n_kv_heads=1, head_size=128),
}


def opened(fields, kv, block=64, seed=7):
    cfg = ol.config(**{**fields, "half_kv": kv})
    tensors, size = ol.places(cfg)
    ck = ol.synth_checkpoint(cfg, tensors, size, seed=seed)
    ol.vary_vectors(cfg, tensors, ck, seed=13)
    ol.sharpen(cfg, tensors, ck, 5.0)
    cos, sin = ol.rope_tables(cfg.seq_len, cfg.head_size, 10000.0)
    return package().open_config(cfg, tensors, ck, cos, sin, max_block=block), cfg, tensors, ck, cos, sin


def tokens(n, vocab=320, seed=3):
    return [1] + [int(t) for t in np.random.default_rng(seed).integers(3, vocab, size=n - 1)]


def rows_of(kv, cfg, count):
    return np.stack([kv[k].reshape(cfg.n_layers, count, cfg.n_kv_heads, cfg.head_size) for k in ("keys", "values")])


@pytest.mark.parametrize("form", sorted(FORMS))
@pytest.mark.parametrize("count", [31, 32, 100, 129])
def test_the_first_layers_cache_is_the_float32_caches_in_8_bits(form, count):
    """the first layer's keys and values do not depend on attention: the float32 cache's rows, quantized"""
    full, cfg, *_ = opened(FORMS[form], 0)
    eight = opened(FORMS[form], 8)[0]
    ids = tokens(count)
    for eng in (full, eight):
        eng.forwardMany(ids, 0)
    want = rows_of(full.keysAndValues(0, count), cfg, count)[:, 0]
    got = rows_of(eight.keysAndValues(0, count), cfg, count)[:, 0]
    model = cl.Model(cfg.n_kv_heads, cfg.head_size, cfg.seq_len)
    model.append(want[0], want[1], 0)
    np.testing.assert_array_equal(got, model.read(0, count, count).astype(np.float32))
    assert eight.memoryBytes() < full.memoryBytes() + (4 << 20)


class Forward:
    """the llama form's forward pass by the oracle's kernels, one token at a time, with the attention over the NumPy cache
    in float64"""

    def __init__(self, cfg, tensors, ck, cos, sin):
        self.c, self.t, self.ck, self.cos, self.sin = cfg, tensors, ck, cos, sin
        self.caches = [cl.Model(cfg.n_kv_heads, cfg.head_size, cfg.seq_len) for _ in range(cfg.n_layers)]
        self.bias = 64 if cfg.relaxed else 0

    def matrix(self, name, layer, rows, k):
        t = self.t[package().T[name]]
        at, sa = t.offset + layer * rows * k, t.scales + layer * rows * (k // 32) * 4
        return (self.ck[at:at + rows * k].view(np.int8).reshape(rows, k),
                np.frombuffer(self.ck[sa:sa + rows * (k // 32) * 4].tobytes(), dtype=np.float32).reshape(rows, -1))

    def vector(self, name, layer, n):
        at = self.t[package().T[name]].offset + 4 * layer * n
        return np.frombuffer(self.ck[at:at + 4 * n].tobytes(), dtype=np.float32)

    def times(self, x, name, layer, rows):
        w, ws = self.matrix(name, layer, rows, x.size)
        return ol.matmul(*ol.quantize_x(x, self.bias), w, ws, rows, x.size, self.bias, 0)[0]

    def rope(self, x, pos):
        p = x.reshape(-1, self.c.head_size // 2, 2)
        out = np.empty_like(p)
        out[..., 0] = p[..., 0] * self.cos[pos] - p[..., 1] * self.sin[pos]
        out[..., 1] = p[..., 0] * self.sin[pos] + p[..., 1] * self.cos[pos]
        return out.reshape(-1)

    def step(self, token, pos):
        c = self.c
        qd, kd = c.n_heads * c.head_size, c.n_kv_heads * c.head_size
        e, es = self.matrix("token_embedding_table", 0, c.vocab_size, c.dim)
        x = (e[token].reshape(-1, 32).astype(np.float32) * es[token][:, None]).reshape(-1)
        for l in range(c.n_layers):
            h = ol.rmsnorm(x, self.vector("rms_att_weight", l, c.dim), c.rms_norm_eps)
            q, k, v = self.times(h, "wq", l, qd), self.times(h, "wk", l, kd), self.times(h, "wv", l, kd)
            q, k = self.rope(q, pos), self.rope(k, pos)
            self.caches[l].append(k[None], v[None], pos)
            out, _ = self.caches[l].attention(q[None], pos, c.n_heads)
            x = x + self.times(out.reshape(-1).astype(np.float32), "wo", l, c.dim)
            h = ol.rmsnorm(x, self.vector("rms_ffn_weight", l, c.dim), c.rms_norm_eps)
            a, b = self.times(h, "w1", l, c.hidden_dim), self.times(h, "w3", l, c.hidden_dim)
            a64 = a.astype(np.float64)
            x = x + self.times((a64 / (1 + np.exp(-a64)) * b).astype(np.float32), "w2", l, c.dim)
        h = ol.rmsnorm(x, self.vector("rms_final_weight", 0, c.dim), c.rms_norm_eps)
        return self.times(h, "token_embedding_table", 0, c.vocab_size)


def test_logits_follow_the_forward_pass_over_the_quantized_cache():
    """against the oracle's kernels with the attention over the NumPy cache: what is left are float32 roundings that now and
    then move an activation to the next of its 63 steps, where the cache moves every key and value: less than a quarter of
    what the cache itself changes, and nothing like it in the first block, where no position is in 8 bits"""
    eight, cfg, tensors, ck, cos, sin = opened(FIELDS, 8)
    full = opened(FIELDS, 0)[0]
    ref, ids = Forward(cfg, tensors, ck, cos, sin), tokens(110)
    apart, own = [], []
    for i, t in enumerate(ids):
        want = ref.step(t, i)
        for eng in (eight, full):
            eng.forward(t, i)
        own.append(np.sqrt(np.mean((eight.logits() - want) ** 2)) / want.std())
        apart.append(np.sqrt(np.mean((full.logits() - want) ** 2)) / want.std())
    own, apart = np.array(own), np.array(apart)
    assert np.mean(own[64:]) < np.mean(apart[64:]) / 4, (own, apart)
    assert np.mean(own[:32]) < np.mean(apart[64:]) / 4
    prompt = opened(FIELDS, 8)[0]
    prompt.forwardMany(ids[:-1], 0)
    prompt.forward(ids[-1], 109)
    assert np.sqrt(np.mean((prompt.logits() - want) ** 2)) / want.std() < np.mean(apart[64:]) / 2


@pytest.mark.parametrize("form", sorted(FORMS))
def test_replayed_steps_equal_eager_ones(form, monkeypatch):
    """the same bits from replayed steps, from eager ones, and from one token at a time through forward()"""
    got = []
    for graph in ("1", "0"):
        monkeypatch.setenv("PYODIDE_LLM_HIP_GRAPH", graph)
        eng = opened(FORMS[form], 8)[0]
        eng.forwardMany(tokens(40)[:-1], 0)
        ids, token, pos = [], tokens(40)[-1], 39
        while len(ids) < 150:
            ids += eng.generateMany(token, pos, [], 0, min(50, 150 - len(ids)), 0.0, 0.9, 1.0, [], [])
            token, pos = ids[-1], 39 + len(ids)
        got.append((ids, np.array(eng.logits()), eng.keysAndValues(0, pos)))
    assert got[0][0] == got[1][0]
    np.testing.assert_array_equal(got[0][1], got[1][1])
    for name in ("keys", "values"):
        np.testing.assert_array_equal(got[0][2][name], got[1][2][name])
    eng = opened(FORMS[form], 8)[0]
    eng.forwardMany(tokens(40)[:-1], 0)
    for i, t in enumerate([tokens(40)[-1]] + got[0][0][:-1]):
        eng.forward(t, 39 + i)
        assert int(np.argmax(eng.logits())) == got[0][0][i]
    np.testing.assert_array_equal(eng.logits(), got[0][1])


def test_steps_after_a_stopped_round_equal_steps_without_one(monkeypatch):
    """a stop token ends a round whose later replays have written rows past it: the positions taken again hold what they
    would have held"""
    ids, randoms = None, [float(r) for r in np.random.default_rng(2).random(40)]
    got = []
    for stop in (False, True):
        eng = opened(FIELDS, 8)[0]
        eng.forwardMany(tokens(20)[:-1], 0)
        if not stop:
            ids = eng.generateMany(tokens(20)[-1], 19, tokens(20), 20, 40, 1.0, 1.0, 1.0, randoms, [])
        else:
            at = max(i for i in range(1, 30) if ids[i] not in ids[:i])
            first = eng.generateMany(tokens(20)[-1], 19, tokens(20), 20, 40, 1.0, 1.0, 1.0, randoms, [ids[at]])
            assert first == ids[:at + 1]
            pos = 19 + len(first)
            kv = eng.keysAndValues(0, pos)
            rest = eng.generateMany(first[-1], pos, tokens(20) + first, pos, 40 - len(first), 1.0, 1.0, 1.0,
                                    randoms[len(first):], [])
            assert first + rest == ids
            plain = opened(FIELDS, 8)[0]
            plain.forwardMany(tokens(20)[:-1], 0)
            for i, t in enumerate([tokens(20)[-1]] + first[:-1]):
                plain.forward(t, 19 + i)
            want = plain.keysAndValues(0, pos)
            for name in kv:
                np.testing.assert_array_equal(kv[name], want[name])
        got.append((np.array(eng.logits()), eng.keysAndValues(0, 59)))
    np.testing.assert_array_equal(got[0][0], got[1][0])
    for name in ("keys", "values"):
        np.testing.assert_array_equal(got[0][1][name], got[1][1][name])


def test_a_turn_taken_again():
    """back to an earlier position: within the latest ones the same bits as a conversation that never went on; further back
    the block's earlier positions by their 8-bit values, finite and close"""
    first, other = tokens(200), tokens(200, seed=9)
    eng = opened(FIELDS, 8)[0]
    eng.forwardMany(first[:150], 0)
    for back, exact in ((100, True), (40, False)):
        eng.forwardMany(other[back:back + 30], back)
        eng.forward(other[back + 30], back + 30)
        fresh = opened(FIELDS, 8)[0]
        fresh.forwardMany((first[:100] if back == 100 else first[:40])[:back], 0)
        fresh.forwardMany(other[back:back + 30], back)
        fresh.forward(other[back + 30], back + 30)
        a, b = np.array(eng.logits()), np.array(fresh.logits())
        if exact:
            assert np.max(np.abs(a - b)) <= 0.25 * b.std()
            ka, kb = (rows_of(x.keysAndValues(0, 131), eng.config, 131)[:, 0] for x in (eng, fresh))
            np.testing.assert_array_equal(ka, kb)
        else:
            assert np.isfinite(a).all() and np.sqrt(np.mean((a - b) ** 2)) < b.std()


def test_a_context_past_the_float32_caches_limit():
    """a context that the ordered attention refuses: opened, filled across its end, replayed"""
    fields = dict(FIELDS, seq_len=45000)
    with pytest.raises(package().HipError):
        opened(fields, 0)
    eng = opened(fields, 8, block=1024)[0]
    ids = tokens(44990)
    for at in range(0, 44989, 1024):
        eng.forwardMany(ids[at:min(44989, at + 1024)], at)
    got = eng.generateMany(ids[-1], 44989, [], 0, 11, 0.0, 0.9, 1.0, [], [])
    assert len(got) == 11 and np.isfinite(eng.logits()).all()
    with pytest.raises(package().HipError):
        eng.forward(1, 45000)


@pytest.mark.parametrize("kv", [0, 1, 8])
@pytest.mark.parametrize("form", ["llama", "gpt2", "qwen int6"])
def test_scores_are_those_of_the_steps_logits(form, kv):
    """he_score's rows against the log softmax in float64 of the logits that forward() gives each token; float32 and float16
    caches give each token's logits to the bit however it is run, and a log probability is then off by 2^-17 at most (its
    sums) and its own rounding. Over 8 bits a token's attention is summed in another order alone or in a prompt: its rows
    are held to those of the same pass"""
    block = 64
    ids = tokens(150)
    eng, cfg = opened(FORMS[form], kv, block)[:2]
    got = eng.score(ids, 0, top=5)
    one = opened(FORMS[form], kv, block)[0]
    worst = 0.0
    for i, t in enumerate(ids):
        one.forward(t, i)
        x = one.logits().astype(np.float64)
        lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
        if i + 1 < len(ids):
            worst = max(worst, abs(got["logp"][i, 0] - lp[ids[i + 1]]))
        if kv != 8:
            assert abs(got["entropy"][i] + (np.exp(lp) * lp).sum()) < 1e-4
            np.testing.assert_array_equal(got["ids"][i], np.argsort(-x, kind="stable")[:5])
            np.testing.assert_allclose(got["logps"][i], lp[got["ids"][i]], atol=2.0 ** -16, rtol=0)
    assert worst <= (2.0 ** -16 if kv != 8 else 0.5), worst
    assert np.isnan(got["logp"][-1, 0])
    assert np.isfinite(got["logps"]).all() and (np.diff(got["logps"], axis=1) <= 0).all()


def test_scores_with_outlier_channels():
    fields = dict(FIELDS, outliers=[3, 17, 40])
    eng, one = opened(fields, 0)[0], opened(fields, 0)[0]
    ids = tokens(20)
    got = eng.score(ids, 0, given=[[5, 6]] * 20)
    for i, t in enumerate(ids):
        one.forward(t, i)
        x = one.logits().astype(np.float64)
        lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
        np.testing.assert_allclose(got["logp"][i], lp[[5, 6]], atol=2.0 ** -16, rtol=0)


def test_log_probabilities_of_the_last_step():
    eng = opened(FIELDS, 0)[0]
    with pytest.raises(package().HipError):
        eng.logprobs(given=[3])  # no step with logits has run
    eng.forwardMany(tokens(10), 0)
    ids = eng.generateMany(5, 10, tokens(10) + [5], 11, 7, 0.0, 0.9, 1.3, [], [])
    x = eng.logits().astype(np.float64)
    lp = x - x.max() - np.log(np.exp(x - x.max()).sum())
    got = eng.logprobs(given=[ids[-1], 0], top=32)
    np.testing.assert_allclose(got["logp"], lp[[ids[-1], 0]], atol=2.0 ** -16, rtol=0)
    assert got["ids"][0] == ids[-1]
    np.testing.assert_array_equal(got["ids"], np.argsort(-x, kind="stable")[:32])
    assert abs(got["entropy"] + (np.exp(lp) * lp).sum()) < 1e-4
    assert eng.logprobs()["logp"].size == 0


def test_scores_that_are_refused():
    pk = package()
    eng, cfg = opened(FIELDS, 8)[:2]
    lib, f = pk.library(), np.zeros(64, dtype=np.float32)
    i = np.array([5, 6], dtype=np.int32)
    ip, fp = ctypes.c_void_p(i.ctypes.data), ctypes.c_void_p(f.ctypes.data)
    E = pk.hip_engine
    for args, code in (((None, 2, 0, ip, 1, 0, fp, fp, None, None), E.HE_E_ARG),
                       ((ip, 0, 0, ip, 1, 0, fp, fp, None, None), E.HE_E_ARG),
                       ((ip, 65, 0, ip, 1, 0, fp, fp, None, None), E.HE_E_ARG),
                       ((ip, 2, 299, ip, 1, 0, fp, fp, None, None), E.HE_E_STATE),
                       ((ip, 2, -1, ip, 1, 0, fp, fp, None, None), E.HE_E_STATE),
                       ((ip, 2, 0, None, 1, 0, fp, fp, None, None), E.HE_E_ARG),
                       ((ip, 2, 0, ip, -1, 0, fp, fp, None, None), E.HE_E_ARG),
                       ((ip, 2, 0, ip, 1, 33, fp, fp, ip, fp), E.HE_E_ARG),
                       ((ip, 2, 0, ip, 1, 2, fp, fp, None, fp), E.HE_E_ARG),
                       ((ip, 2, 0, None, 0, 0, None, None, None, None), E.HE_E_ARG)):
        assert lib.he_score(eng._h, *args) == code
    i[0] = 320
    assert lib.he_score(eng._h, ip, 2, 0, ip, 1, 0, fp, fp, None, None) == E.HE_E_ARG
    assert lib.he_score(None, ip, 2, 0, ip, 1, 0, fp, fp, None, None) == E.HE_E_ARG
    assert lib.he_logprobs(None, ip, 1, 0, fp, fp, None, None) == E.HE_E_ARG


@pytest.mark.skipif(shutil.which("node") is None, reason="no node here")
def test_the_node_host_gives_the_same(tmp_path):
    """forward_hip.mjs with eightBitCache, score() and logprobs(): the Python host's numbers to the bit"""
    eng, cfg, tensors, ck, cos, sin = opened(FIELDS, 8)
    ids = tokens(90)
    ck.tofile(tmp_path / "checkpoint.bin")
    np.asarray(cos, np.float32).tofile(tmp_path / "cos.bin")
    np.asarray(sin, np.float32).tofile(tmp_path / "sin.bin")
    job = {"size": int(ck.size), "plan": {**plan_of(cfg, tensors), "half_kv": True}, "tokens": ids, "steps": 20}
    (tmp_path / "job.json").write_text(json.dumps(job))
    proc = subprocess.run(["node", os.path.join(REPO, "tests", "node", "score_engine.mjs"), str(tmp_path / "job.json")],
                          stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=120)
    assert proc.returncode == 0, proc.stderr[-3000:]
    out = json.loads(proc.stdout.strip().splitlines()[-1])
    got = eng.score(ids, 0, top=3)
    steps = eng.generateMany(7, 90, [], 0, 16, 0.0, 0.9, 1.0, [], [])
    last = eng.logprobs(given=[steps[-1], 3], top=2)
    assert out["steps"] == steps
    for name in ("entropy", "ids", "logps"):
        np.testing.assert_array_equal(np.array(out["score"][name], dtype=np.float32),
                                      got[name].reshape(-1).astype(np.float32))
    np.testing.assert_array_equal(np.array(out["score"]["logp"][:-1], dtype=np.float32), got["logp"][:-1, 0])
    assert out["score"]["logp"][-1] is None  # (NaN)
    np.testing.assert_array_equal(np.array(out["last"]["logp"], dtype=np.float32), last["logp"])
    np.testing.assert_array_equal(out["last"]["ids"], last["ids"])
    assert out["threw"] == [True] * 4
    assert out["footprint"] + ck.size >= out["memoryBytes"]


@pytest.mark.parametrize("form", ["llama", "qwen int6", "wide heads"])
@pytest.mark.parametrize("start", [30, 1400])
def test_replayed_steps_over_a_long_cache_equal_eager_ones(form, start, monkeypatch):
    """a cache past the one-launch form: a step's parts are those of its position, whether the launch knows it or not"""
    fields, got = dict(FORMS[form], seq_len=3000), []
    for graph in ("1", "0"):
        monkeypatch.setenv("PYODIDE_LLM_HIP_GRAPH", graph)
        eng = opened(fields, 8, block=512)[0]
        text = tokens(start + 1)
        for at in range(0, start, 512):
            eng.forwardMany(text[at:min(start, at + 512)], at)
        randoms = [float(r) for r in np.random.default_rng(4).random(48)]
        ids = eng.generateMany(text[-1], start, text, start + 1, 48, 1.0, 1.0, 1.0, randoms, [])
        got.append((ids, np.array(eng.logits()), eng.keysAndValues(start, len(ids))))
    assert len(got[0][0]) == 48 and got[0][0] == got[1][0]
    np.testing.assert_array_equal(got[0][1], got[1][1])
    for name in ("keys", "values"):
        np.testing.assert_array_equal(got[0][2][name], got[1][2][name])


def run_one_by_one(eng, ids, start=0):
    for i, t in enumerate(ids):
        eng.forward(t, start + i)


@pytest.mark.parametrize("back", [0, 10, 33, 39])
def test_a_look_back_leaves_the_rows_behind_it(back):
    """a token run again at an earlier position (for its logits), then the conversation's next one: as without the look back"""
    ids = tokens(60)
    plain, eng = opened(FIELDS, 8)[0], opened(FIELDS, 8)[0]
    for e in (plain, eng):
        run_one_by_one(e, ids[:40])
    eng.forward(ids[back], back)
    for e in (plain, eng):
        run_one_by_one(e, ids[40:], 40)
    np.testing.assert_array_equal(eng.logits(), plain.logits())
    a, b = (e.keysAndValues(0, 60) for e in (eng, plain))
    for name in a:
        np.testing.assert_array_equal(a[name], b[name])


def first_layer(eng, count):
    return rows_of(eng.keysAndValues(0, count), eng.config, count)[:, 0]


def test_a_return_from_far_back_finds_the_last_block():
    """far back and forward to the end again: the block that was being filled stands as its 8-bit values, not as zeros"""
    ids = tokens(210)
    eng, full = opened(FIELDS, 8)[0], opened(FIELDS, 0)[0]
    for e in (eng, full):
        run_one_by_one(e, ids[:200])
        e.forward(ids[10], 10)
        run_one_by_one(e, ids[200:], 200)
    want = rows_of(full.keysAndValues(0, 210), full.config, 210)[:, 0]
    model = cl.Model(2, 16, 300)
    model.append(want[0, :200], want[1, :200], 0)
    # the first block, its rows from 8 bits but the one run again, is quantized anew
    again = model.read(0, 32, 1 << 40).astype(np.float32)
    again[:, 10] = want[:, 10]
    model.append(again[0], again[1], 0)
    zeros = np.zeros((24, 2, 16), dtype=np.float32)
    model.append(zeros, zeros, 200)
    model.rewind(200)
    model.append(want[0, 200:], want[1, 200:], 200)
    np.testing.assert_array_equal(first_layer(eng, 210), model.read(0, 210, 210).astype(np.float32))


@pytest.mark.parametrize("pos", [12, 31, 32, 50, 140])
def test_positions_passed_over_stand_as_zeros(pos):
    """as in the float32 cache"""
    ids = tokens(20)
    eng, full = opened(FIELDS, 8)[0], opened(FIELDS, 0)[0]
    for e in (eng, full):
        run_one_by_one(e, ids[:10])
        run_one_by_one(e, ids[10:], pos)
    n = pos + 10
    want = rows_of(full.keysAndValues(0, n), full.config, n)[:, 0]
    assert (want[:, 10:pos] == 0).all()
    model = cl.Model(2, 16, 300)
    model.append(want[0], want[1], 0)
    np.testing.assert_array_equal(first_layer(eng, n), model.read(0, n, n).astype(np.float32))


def test_a_position_run_again_with_another_token_is_read_so():
    """another token at an earlier position, then the conversation's next one: every later token reads the new row, as over
    the float32 cache, whether the position's block is still held in float32 (100) or not (10)"""
    ids = tokens(190)
    for at in (100, 10):
        eng, full = opened(FIELDS, 8)[0], opened(FIELDS, 0)[0]
        for e in (eng, full):
            run_one_by_one(e, ids[:180])
            e.forward(7, at)
            run_one_by_one(e, ids[180:], 180)
        want = rows_of(full.keysAndValues(0, 190), full.config, 190)[:, 0]
        got = first_layer(eng, 190)
        first = at // 32 * 32
        steps = np.abs(want[:, first:first + 32]).max((1, 3), keepdims=True) / 127
        assert (np.abs(got[:, first:first + 32] - want[:, first:first + 32]) <= 1.01 * steps).all()
        old = rows_of(opened_after(ids[:180]).keysAndValues(0, 180), full.config, 180)[:, 0]
        assert (np.abs(old[:, at] - want[:, at]) > 2 * steps[:, 0]).any()


def opened_after(ids):
    eng = opened(FIELDS, 8)[0]
    run_one_by_one(eng, ids)
    return eng


@pytest.mark.parametrize("seed", range(40))
def test_calls_at_any_positions_leave_the_rows_last_written(seed):
    """calls here and there, far back and past the end: the first layer's cache is the float32 cache's but for roundings to 8
    bits. A block is quantized at most once more than calls have touched it, each time off by half a step, at most 1 / 127 of
    the head's largest value so far (another scale moves values that have been rounded before)"""
    rng = np.random.default_rng(seed)
    eng, full = opened(FIELDS, 8)[0], opened(FIELDS, 0)[0]
    end = furthest = 0
    largest, touched = np.zeros((2, 1, 2, 1)), np.ones(300 // 32 + 1)

    def agree(n):
        nonlocal largest
        want = rows_of(full.keysAndValues(0, 300), full.config, 300)[:, 0]
        largest = np.maximum(largest, np.abs(want).max((1, 3), keepdims=True))
        got = rows_of(eng.keysAndValues(0, n), eng.config, n)[:, 0]
        off = 0.501 * touched[np.arange(n) // 32][None, :, None, None] * largest / 127
        assert (np.abs(got - want[:, :n]) <= off).all()

    for _ in range(25):
        pos = [end, int(rng.integers(0, furthest + 1)), max(0, end - int(rng.integers(0, 130))), furthest,
               furthest + int(rng.integers(0, 60))][int(rng.choice(5, p=[0.3, 0.25, 0.25, 0.1, 0.1]))]
        count = min(int(rng.choice([1, 1, 1, 3, 20, 64])), 280 - pos)
        if count < 1:
            continue
        ids = [int(t) for t in rng.integers(3, 320, size=count)]
        for e in (eng, full):
            e.forwardMany(ids, pos) if count > 1 else e.forward(ids[0], pos)
        end = pos + count
        furthest = max(furthest, end)
        touched[pos // 32:end // 32 + 1] += 1
        agree(end)
    for e in (eng, full):
        e.forward(5, furthest)
    agree(furthest + 1)


@pytest.mark.parametrize("count", [20, 140, 160])
def test_rows_behind_the_end_are_no_other_positions(count):
    """keysAndValues past the last token: zeros where no token has been, as the float32 cache's"""
    eng = opened(FIELDS, 8)[0]
    eng.forwardMany(tokens(count)[:64], 0)
    for at in range(64, count, 64):
        eng.forwardMany(tokens(count)[at:at + 64], at)
    got = rows_of(eng.keysAndValues(0, 200), eng.config, 200)
    assert (got[:, :, count:] == 0).all()
    kv = rows_of(eng.keysAndValues(0, count), eng.config, count)
    np.testing.assert_array_equal(got[:, :, :count], kv)
    inside = rows_of(eng.keysAndValues(count - 5, 20), eng.config, 20)
    np.testing.assert_array_equal(inside, got[:, :, count - 5:count + 15])
    beyond = eng.keysAndValues(count + 3, 9)
    assert all((beyond[name] == 0).all() for name in beyond)


@pytest.mark.parametrize("kv", [0, 8])
def test_steps_before_the_first_position_are_refused(kv):
    """by replayed steps too, whose position only the device looks at"""
    eng = opened(FIELDS, kv)[0]
    eng.forwardMany(tokens(5), 0)
    assert len(eng.generateMany(7, 5, [], 0, 6, 0.0, 0.9, 1.0, [], [])) == 6  # (from here on steps are replayed)
    for pos in (-1, -64, -2147483648):
        with pytest.raises(package().HipError):
            eng.generateMany(7, pos, [], 0, 6, 0.0, 0.9, 1.0, [], [])
    assert len(eng.generateMany(7, 11, [], 0, 6, 0.0, 0.9, 1.0, [], [])) == 6


def distribution(x):
    x = x.astype(np.float64)
    return x - x.max(-1, keepdims=True) - np.log(np.exp(x - x.max(-1, keepdims=True)).sum(-1, keepdims=True))


def held_together(got, lp, given, top):
    """score()'s rows against the rows' whole distributions lp (float64, each off by 2^-16 at most)"""
    np.testing.assert_allclose(got["logp"], np.take_along_axis(lp, given, 1), atol=2.0 ** -15, rtol=0)
    np.testing.assert_allclose(got["entropy"], -(np.exp(lp) * lp).sum(-1), atol=1e-3, rtol=0)
    order = np.argsort(-lp, axis=1, kind="stable")[:, :top]
    np.testing.assert_allclose(got["logps"], np.take_along_axis(lp, order, 1), atol=2.0 ** -15, rtol=0)
    np.testing.assert_allclose(np.take_along_axis(lp, got["ids"].astype(np.int64), 1), got["logps"], atol=2.0 ** -15, rtol=0)
    assert all(len(set(row)) == top for row in got["ids"].tolist())


@pytest.mark.parametrize("form", sorted(FORMS))
def test_scores_over_8_bits_are_of_one_pass(form):
    """every output of a pass over 8 bits against the log probabilities of the whole vocabulary that the same pass gives; and
    the distributions near the steps' own (a row of another token lies ten times as far)"""
    ids = tokens(150)
    vocab = np.tile(np.arange(320), (150, 1))
    lp = opened(FORMS[form], 8)[0].score(ids, 0, given=vocab)["logp"].astype(np.float64)
    np.testing.assert_allclose(np.exp(lp).sum(1), 1.0, atol=1e-4)
    given = np.random.default_rng(1).integers(0, 320, (150, 3))
    held_together(opened(FORMS[form], 8)[0].score(ids, 0, given=given, top=7), lp, given, 7)
    text = opened(FORMS[form], 8)[0].score(ids, 0, top=7)
    held_together({n: x[:-1] for n, x in text.items()}, lp[:-1], np.array(ids[1:])[:, None], 7)
    assert np.isnan(text["logp"][-1, 0])
    one = opened(FORMS[form], 8)[0]
    steps = []
    for i, t in enumerate(ids):
        one.forward(t, i)
        steps.append(distribution(one.logits()))
    steps = np.array(steps)
    near = np.sqrt(np.mean((steps - lp) ** 2, 1))
    for shift in (1, 2, 7):
        assert near.max() < np.sqrt(np.mean((steps[shift:] - lp[:-shift]) ** 2, 1)).min()


def test_one_tokens_scores_over_8_bits_are_its_steps():
    """a pass of one token is the step that forward() runs: its log probabilities are those of the step's logits"""
    ids = tokens(120)
    eng, one = opened(FIELDS, 8)[0], opened(FIELDS, 8)[0]
    for i, t in enumerate(ids):
        one.forward(t, i)
        got, lp = eng.score([t], i, given=[[5, 9]], top=4), distribution(one.logits())[None]
        held_together(got, lp, np.array([[5, 9]]), 4)


@pytest.mark.parametrize("kv", [0, 8])
def test_scores_of_a_long_text_and_a_large_vocabulary(kv):
    """more tokens than a pass runs and than logits are held at once; rows in several parts; fewer tokens asked about first, so
    that what holds them grows: every output of every row"""
    fields = dict(FIELDS, vocab_size=9001, seq_len=1500)
    eng, cfg = opened(fields, kv, 2048)[:2]
    few = eng.score(tokens(3, 9001), 0, top=2)
    ids = tokens(1400, 9001, seed=5)
    given = np.random.default_rng(2).integers(0, 9001, (1400, 2))
    got = eng.score(ids, 0, given=given, top=6)
    if kv == 0:
        one, lp = opened(fields, 0)[0], []
        for i, t in enumerate(ids):
            one.forward(t, i)
            lp.append(distribution(one.logits()))
        held_together(got, np.array(lp), given, 6)
    else:
        # the same pass again, asked for a part of the vocabulary: what it shares with the first is the same to the bit
        again = eng.score(ids, 0, given=got["ids"], top=0)
        np.testing.assert_array_equal(again["logp"], got["logps"])
        np.testing.assert_array_equal(again["entropy"], got["entropy"])
        full = opened(fields, 0, 2048)[0].score(ids, 0, given=given, top=6)
        assert np.mean(np.abs(full["logp"] - got["logp"])) < 0.05 < np.mean(np.abs(full["logp"][1:] - got["logp"][:-1]))
        assert np.mean(full["ids"][:, 0] == got["ids"][:, 0]) > 0.9
    assert few["ids"].shape == (3, 2)


@pytest.mark.parametrize("form", sorted(FORMS))
def test_a_turn_taken_again_is_the_turn_itself(form):
    """back within the latest positions, once and twice: the logits and the cache of a conversation that was split the same way
    and never went on, to the bit"""
    first, other, third = tokens(150), tokens(150, seed=9), tokens(150, seed=10)
    eng, plain = (opened(FORMS[form], 8)[0] for _ in range(2))
    for e in (eng, plain):
        e.forwardMany(first[:60], 0)
        e.forwardMany(first[60:100], 60)
    eng.forwardMany(first[100:150], 100)
    for at, ids in ((100, other), (70, third)):
        for e in (eng, plain):
            if at == 100 or e is eng:
                e.forwardMany(ids[:30], at)
                e.forward(ids[30], at + 30)
        if at == 70:
            plain = opened(FORMS[form], 8)[0]
            plain.forwardMany(first[:60], 0)
            plain.forwardMany(first[60:70], 60)
            plain.forwardMany(ids[:30], at)
            plain.forward(ids[30], at + 30)
        if at == 100:
            np.testing.assert_array_equal(eng.logits(), plain.logits())
            a, b = (e.keysAndValues(0, at + 31) for e in (eng, plain))
            for name in a:
                np.testing.assert_array_equal(a[name], b[name])
        else:  # (positions 60..69 came with another split: the same keys and values in the first layer)
            np.testing.assert_array_equal(*(rows_of(e.keysAndValues(0, 101), e.config, 101)[:, 0] for e in (eng, plain)))


WIDE = dict(dim=1024, hidden_dim=2048, n_layers=2, n_heads=8, n_kv_heads=2, head_size=128, vocab_size=2000, seq_len=1200,
            shared_classifier=1)


def attention32(cache, q, pos, nh):
    """cl.Model.attention of one token in NumPy's float32"""
    hs, first = cache.hs, pos // cl.BLOCK
    q = q.reshape(nh, hs).astype(np.float32)
    k, v = (np.concatenate([cache.eight(w, b) for b in range(first)] + [cache.rows[w, first * cl.BLOCK:pos + 1]]).astype(np.float32)
            for w in range(2))
    out = np.zeros((1, nh, hs))
    for h in range(nh):
        g = h // (nh // cache.nkv)
        s = k[:, g] @ q[h] / np.float32(np.sqrt(hs))
        e = np.exp(s - s.max())
        out[0, h] = e @ v[:, g] / e.sum()
    return out, None


@pytest.mark.parametrize("fields", [WIDE, dict(WIDE, dim=2048, n_heads=16, n_kv_heads=8),
                                    dict(WIDE, n_heads=4, n_kv_heads=4, head_size=256)])
def test_wider_models(fields, monkeypatch):
    """the first layer's cache exactly; logits as near to the oracle's kernels with the attention over the NumPy cache in float64
    as with that attention in NumPy's float32 (twice as far at most: both are float32 roundings that move an activation to the
    next of its steps, more of them the wider a layer is); replayed steps equal to eager ones to the bit"""
    ids = tokens(1000, 2000)
    full, cfg = opened(fields, 0, 1024)[:2]
    eight, _, tensors, ck, cos, sin = opened(fields, 8, 1024)
    for e in (full, eight):
        e.forwardMany(ids, 0)
    want = rows_of(full.keysAndValues(0, 1000), cfg, 1000)[:, 0]
    model = cl.Model(cfg.n_kv_heads, cfg.head_size, cfg.seq_len)
    model.append(want[0], want[1], 0)
    np.testing.assert_array_equal(rows_of(eight.keysAndValues(0, 1000), cfg, 1000)[:, 0],
                                  model.read(0, 1000, 1000).astype(np.float32))
    ref, other = (Forward(cfg, tensors, ck, cos, sin) for _ in range(2))
    for cache in other.caches:
        cache.attention = lambda q, pos, nh, cache=cache: attention32(cache, q, pos, nh)
    own, inherent, prompts = [], [], []
    for i, t in enumerate(ids[:110]):
        want = ref.step(t, i)
        eight.forward(t, i)
        for x, off in ((eight.logits(), own), (other.step(t, i), inherent)):
            off.append(np.sqrt(np.mean((x - want) ** 2)) / want.std())
        if i >= 100:
            prompt = opened(fields, 8, 1024)[0]
            prompt.forwardMany(ids[:i], 0)
            prompt.forward(t, i)
            prompts.append(np.sqrt(np.mean((prompt.logits() - want) ** 2)) / want.std())
    assert np.mean(own[32:]) < 2 * np.mean(inherent[32:]), (np.mean(own[32:]), np.mean(inherent[32:]))
    assert np.mean(prompts) < 2 * np.mean(inherent[32:])
    got = []
    for graph in ("1", "0"):
        monkeypatch.setenv("PYODIDE_LLM_HIP_GRAPH", graph)
        eng = opened(fields, 8, 1024)[0]
        eng.forwardMany(ids[:-1], 0)
        got.append((eng.generateMany(ids[-1], 999, [], 0, 60, 0.0, 0.9, 1.0, [], []), np.array(eng.logits())))
    assert got[0][0] == got[1][0]
    np.testing.assert_array_equal(got[0][1], got[1][1])


def test_scores_at_the_end_of_a_long_text_follow_the_float32_caches():
    """40,000 positions behind the tokens, nearly as many as the ordered attention takes"""
    n, ids = 40000, tokens(40200)
    full, eight = opened(dict(FIELDS, seq_len=40400), 0, 1024)[0], opened(dict(FIELDS, seq_len=45000), 8, 1024)[0]
    lp = []
    for e in (full, eight):
        for at in range(0, n, 1024):
            e.forwardMany(ids[at:min(n, at + 1024)], at)
        lp.append(e.score(ids[n:], n, given=[[5, 9, 77, 200]] * 200)["logp"])
    assert np.sqrt(np.mean((lp[0] - lp[1]) ** 2)) < 0.1 * np.sqrt(np.mean((lp[0][1:] - lp[1][:-1]) ** 2))
