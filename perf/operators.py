"""The operators over a cache held in 8 bits, and the log probabilities of tokens: what a program gives hk_cache_append,
hk_cache_attention and hk_logprobs. A case is a dict of plain values; `listed` names the fixed ones, `draw` makes more of
the same ranges, `prepare` is what a program holds before the call, `run` is the call (in its plain form by elementary
torch operations, or with `own` through the library), `work` its unavoidable bytes and operations, `exact` the same
result in 64 bits.

The cache (one layer's): blocks of 32 positions. A block that is complete holds int8 values with one float32 scale a
kv head for its keys and one for its values, s = f32(max |x| / 127), q = x / s rounded to the nearest (ties to even);
the block being filled, and the latest 128 positions, are kept in float32 besides. A token at position p attends to the
positions before its own block (32 * floor(p / 32)) by their 8-bit values and to those of its own block, up to p, by
their float32 rows.
"""
import ctypes
import importlib
import math

import torch

own = False

BLOCK, RECENT = 32, 128

# query heads, kv heads and head sizes: the repository's own models and tests, and two generic layouts (wide heads, an
# odd group)
HEADS = {
    "llama3-8b": (32, 8, 128),
    "qwen25-7b": (28, 4, 128),
    "llm150m": (8, 8, 64),
    "stories15m": (6, 6, 48),
    "gpt2-small": (12, 12, 64),
    "test-16": (4, 2, 16),
    "test-96": (12, 4, 96),
    "wide-256": (16, 8, 256),
    "odd-32": (10, 5, 32),
}
VOCABS = [320, 32000, 50257, 99487, 128256, 152064]


def listed():
    return [
        # a layer of a 2048-token prompt enters the cache (64 whole blocks)
        dict(name="append-prompt", kind="append", heads="llama3-8b", pos=0, count=2048),
        # a decode step's token, the last of its block: the smallest call, and the one that quantizes
        dict(name="append-token", kind="append", heads="llama3-8b", pos=4095, count=1),
        # one token of an answer after a few thousand tokens, as each decode step and layer calls it
        dict(name="token-4k", kind="attention", heads="llama3-8b", pos=4077, count=1),
        # an answer deep in a long context, seven query heads a kv head
        dict(name="token-32k", kind="attention", heads="qwen25-7b", pos=32001, count=1),
        # a context past what the float32 cache's attention takes
        dict(name="token-131k", kind="attention", heads="llama3-8b", pos=131077, count=1),
        # the smallest model's step: launches and latency
        dict(name="token-15m", kind="attention", heads="stories15m", pos=200, count=1),
        # a prompt block from the start
        dict(name="prompt-2048", kind="attention", heads="llama3-8b", pos=0, count=2048),
        # the next message of a conversation, neither end on a block's edge
        dict(name="turn-37", kind="attention", heads="llama3-8b", pos=1500, count=37),
        # a document's piece far into a long context
        dict(name="prompt-long", kind="attention", heads="qwen25-7b", pos=20003, count=1001),
        # the token just drawn, with twenty alternatives, as a serving call reports them
        dict(name="logprobs-token", kind="logprobs", rows=1, vocab=128256, given=1, top=20, pad=0, banned=False),
        # scoring a text: a block of tokens at once
        dict(name="logprobs-512", kind="logprobs", rows=512, vocab=128256, given=1, top=5, pad=0, banned=False),
        # an odd vocabulary (rows start at any float), half its tokens banned (minus infinity), four answers compared
        dict(name="logprobs-odd", kind="logprobs", rows=200, vocab=50257, given=4, top=20, pad=0, banned=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "logprobs"])
    if kind == "logprobs":
        vocab = rng.choice(VOCABS + [_log_int(rng, 64, 200000)])
        return dict(kind=kind, rows=_log_int(rng, 1, min(1024, 512 * 128256 // vocab)), vocab=vocab,
                    given=rng.choice([1, 1, 2, 4]), top=rng.choice([0, 1, 5, 20, 32]), pad=rng.choice([0, 0, 1, 64]),
                    banned=rng.random() < 0.3)
    heads = rng.choice(sorted(HEADS))
    if kind == "append":
        # (a pass is repeated on the same state, as a turn taken again: a start inside a block goes with a piece that
        # leaves the block's earlier rows among the latest 128)
        if rng.random() < 0.5:
            return dict(kind=kind, heads=heads, pos=_log_int(rng, 1, 60000) - 1, count=_log_int(rng, 1, 96))
        return dict(kind=kind, heads=heads, pos=BLOCK * (_log_int(rng, 1, 1000) - 1), count=_log_int(rng, 2, 2048))
    if rng.random() < 0.5:
        return dict(kind=kind, heads=heads, pos=_log_int(rng, 1, 131072) - 1, count=1)
    count = _log_int(rng, 2, 2048)
    longest = max(1, min(32768, 18_000_000 // count))
    return dict(kind=kind, heads=heads, pos=_log_int(rng, 1, longest) - 1, count=count)


# ---- what a program holds before the call


def _package():
    return importlib.import_module("pyodide-llm_amd")


def _generator(seed, stream):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + stream) % (1 << 62))


def _randn(shape, seed, stream):
    return torch.randn(shape, device="cuda", generator=_generator(seed, stream))


def _quantized(rows):
    """rows [blocks * 32, heads, size] float32 -> int8 [heads, blocks, 32, size], scales [heads, blocks]"""
    n, heads, size = rows.shape
    x = rows.reshape(n // BLOCK, BLOCK, heads, size).permute(2, 0, 1, 3)
    scale = x.abs().amax((2, 3)) / 127.0
    wide = scale.double()[..., None, None]
    q = torch.where(wide > 0, torch.round(x.double() / torch.where(wide > 0, wide, 1.0)), 0.0)
    return q.to(torch.int8), scale


def _slots():
    """where a block's position lies in a value row: the half (0 or 1) and the byte of its sixteen"""
    t = torch.arange(BLOCK, device="cuda")
    return (t >> 2 & 1) * 16 + (t >> 4) * 8 + (t >> 3 & 1) * 4 + (t & 3)


def _prepare_cache(case, seed, filled):
    """the cache with positions 0..filled-1 in it (those of whole blocks in 8 bits, the latest 128 in float32), and the
    rows from the first of the block that `pos` lies in on"""
    nh, nkv, size = HEADS[case["heads"]]
    pos, end = case["pos"], case["pos"] + case["count"]
    blocks = -(-end // BLOCK)
    keys = torch.zeros(nkv, blocks, size // 16, BLOCK, 16, dtype=torch.int8, device="cuda")
    values = torch.zeros(nkv, blocks, size, BLOCK, dtype=torch.uint8, device="cuda")
    scales = torch.zeros(nkv, blocks, 2, device="cuda")
    recent = [torch.zeros(RECENT + BLOCK, nkv, size, device="cuda") for _ in range(2)]
    first = pos // BLOCK * BLOCK
    # keys with strong and weak channels and values around zero, as projections give them
    channel = torch.exp(0.5 * _randn((nkv, size), seed, 1))
    latest = []
    for which in range(2):
        pieces = []
        for at in range(0, end, 16384):  # a piece at a time: the rows of a long context are not held in float32
            n = min(16384, blocks * BLOCK - at)
            rows = _randn((n, nkv, size), seed, 2 + 2 * at + which)
            if which == 0:
                rows *= channel
            pieces.append(rows[max(0, min(first, end - RECENT) - at):max(0, end - at)].clone())
            whole = min(n, max(0, filled // BLOCK * BLOCK - at)) // BLOCK
            if whole:
                q, s = _quantized(rows[:whole * BLOCK])
                b = at // BLOCK
                if which == 0:
                    keys[:, b:b + whole] = q.reshape(nkv, whole, BLOCK, size // 16, 16).transpose(2, 3)
                else:
                    stored = torch.empty(nkv, whole, size, BLOCK, dtype=torch.uint8, device="cuda")
                    stored[..., _slots()] = (q.transpose(2, 3).to(torch.int16) + 128).to(torch.uint8)
                    values[:, b:b + whole] = stored
                scales[:, b:b + whole, which] = s
        rows = torch.cat(pieces)
        at = torch.arange(end - rows.shape[0], end, device="cuda")
        kept = (at >= filled - RECENT) & (at < filled)
        recent[which][at[kept] % RECENT] = rows[kept]
        if end > first + RECENT:  # a piece that has displaced them: the earlier rows of the first block stand apart
            earlier = (at >= first) & (at < pos)
            recent[which][RECENT + at[earlier] - first] = rows[earlier]
        latest.append(rows[pos - end:].reshape(-1, nkv * size).contiguous())
    return dict(case=case, keys=keys, values=values, scales=scales, recent_keys=recent[0], recent_values=recent[1],
                k=latest[0], v=latest[1], nh=nh, nkv=nkv, size=size, handle=None)


def prepare(case, seed):
    if case["kind"] == "logprobs":
        rows, vocab = case["rows"], case["vocab"]
        x = _randn((rows, vocab + case["pad"]), seed, 1) * 2.0
        # a trained model's rows: some flat, some with a few tokens far above the rest
        lift = torch.rand((rows, 8), device="cuda", generator=_generator(seed, 2)) * 14.0
        at = torch.randint(0, vocab, (rows, 8), device="cuda", generator=_generator(seed, 3))
        x.scatter_add_(1, at, lift)
        if case["banned"]:
            x[torch.rand(x.shape, device="cuda", generator=_generator(seed, 4)) < 0.5] = -math.inf
        given = torch.randint(0, vocab, (rows, case["given"]), device="cuda", generator=_generator(seed, 5))
        given[::2, 0] = at[::2, 0]
        state = dict(case=case, logits=x, given=given.to(torch.int32),
                     logp=torch.empty(rows, case["given"], device="cuda"), entropy=torch.empty(rows, device="cuda"),
                     ids=torch.empty(rows, case["top"], dtype=torch.int32, device="cuda"),
                     logps=torch.empty(rows, case["top"], device="cuda"), workspace=None)
        return state
    end = case["pos"] + case["count"]
    if case["kind"] == "append":
        state = _prepare_cache(case, seed, case["pos"])
        state["out"] = [torch.empty_like(state["k"]), torch.empty_like(state["v"])]
        return state
    state = _prepare_cache(case, seed, end)
    state["q"] = _randn((case["count"], state["nh"] * state["size"]), seed, 0) * 1.5
    state["out"] = torch.empty_like(state["q"])
    return state


# ---- the call


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attention": _own_attention, "logprobs": _own_logprobs}[kind](state)
    return {"append": _plain_append, "attention": _plain_attention, "logprobs": _plain_logprobs}[kind](state)


def _handle(state):
    """the hk_cache over the state's buffers and a workspace, made once, as a program keeps them"""
    if state["handle"] is None:
        pk, case = _package(), state["case"]
        cache = pk.HkCache(keys=state["keys"].data_ptr(), values=state["values"].data_ptr(),
                           scales=state["scales"].data_ptr(), recent_keys=state["recent_keys"].data_ptr(),
                           recent_values=state["recent_values"].data_ptr(), n_kv_heads=state["nkv"],
                           head_size=state["size"], seq_len=state["keys"].shape[1] * BLOCK)
        need = pk.library().hk_cache_workspace(ctypes.byref(cache), state["nh"], case["count"])
        space = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        state["handle"] = (pk.library(), pk.hip_engine.check, ctypes.byref(cache), space, need)
    return state["handle"]


def _own_append(state):
    lib, check, cache, _, _ = _handle(state)
    case, width = state["case"], state["nkv"] * state["size"]
    stream = torch.cuda.current_stream().cuda_stream
    keys, values = state["out"]
    check(lib.hk_cache_append(cache, state["k"].data_ptr(), state["v"].data_ptr(), width, case["count"], case["pos"],
                              stream))
    # the rows as the values they now stand for
    check(lib.hk_cache_read(keys.data_ptr(), values.data_ptr(), cache, case["pos"], case["count"],
                            case["pos"] + case["count"], stream))
    return {"keys": keys, "values": values}


def _own_attention(state):
    lib, check, cache, space, need = _handle(state)
    case, width, out = state["case"], state["nkv"] * state["size"], state["out"]
    check(lib.hk_cache_attention(out.data_ptr(), state["q"].data_ptr(), state["k"].data_ptr(), state["v"].data_ptr(),
                                 cache, state["nh"], state["nh"] * state["size"], width, state["nh"] * state["size"],
                                 case["count"], case["pos"], space.data_ptr(), need,
                                 torch.cuda.current_stream().cuda_stream))
    return out


def _own_logprobs(state):
    pk, case = _package(), state["case"]
    lib, top = pk.library(), case["top"]
    if state["workspace"] is None:
        need = lib.hk_logprobs_workspace(case["rows"], case["vocab"], top)
        state["workspace"] = (torch.empty(max(1, need), dtype=torch.uint8, device="cuda"), need)
    space, need = state["workspace"]
    pk.hip_engine.check(lib.hk_logprobs(
        state["logp"].data_ptr(), state["entropy"].data_ptr(), state["ids"].data_ptr() if top else None,
        state["logps"].data_ptr() if top else None, state["logits"].data_ptr(), state["logits"].stride(0),
        state["given"].data_ptr(), case["given"], case["rows"], case["vocab"], top, space.data_ptr(), need,
        torch.cuda.current_stream().cuda_stream))
    return _outputs(state["logp"], state["entropy"], state["ids"], state["logps"], top)


def _outputs(logp, entropy, ids, logps, top):
    got = {"logp": logp, "entropy": entropy}
    return {**got, "ids": ids, "logps": logps} if top else got


def _own_block_rows(state, which):
    """the float32 rows from the first of pos's block on: the earlier ones from the cache, then the call's"""
    case, recent = state["case"], state["recent_" + ("keys", "values")[which]]
    pos, first = case["pos"], case["pos"] // BLOCK * BLOCK
    at = torch.arange(first, pos, device="cuda")
    displaced = pos + case["count"] > first + RECENT and case["kind"] == "attention"
    earlier = recent[RECENT + at - first] if displaced else recent[at % RECENT]
    return torch.cat([earlier, state["kv"[which]].reshape(-1, state["nkv"], state["size"])])


def _plain_append(state):
    case = state["case"]
    pos, first, end = case["pos"], case["pos"] // BLOCK * BLOCK, case["pos"] + case["count"]
    whole = end // BLOCK * BLOCK - first
    got = {}
    for which, name in enumerate(("keys", "values")):
        rows = _own_block_rows(state, which)
        if whole > 0:
            x = rows[:whole].reshape(whole // BLOCK, BLOCK, state["nkv"], state["size"])
            scale = x.abs().amax((1, 3), keepdim=True) / 127.0
            wide = scale.double()  # (values next to a rounding's border)
            q = torch.where(wide > 0, torch.round(x.double() / torch.where(wide > 0, wide, 1.0)), 0.0).float()
            rows = torch.cat([(q * scale).reshape(whole, state["nkv"], state["size"]), rows[whole:]])
        got[name] = rows[pos - first:].reshape(case["count"], -1)
    return got


def _plain_attention(state):
    case, nh, nkv, size = state["case"], state["nh"], state["nkv"], state["size"]
    pos, count = case["pos"], case["count"]
    first, old = pos // BLOCK * BLOCK, (pos + count - 1) // BLOCK  # (old: the 8-bit blocks that any token sees)
    scale_k, scale_v = state["scales"][:, :old, None, None].unbind(-1)
    k8 = state["keys"][:, :old].transpose(2, 3).reshape(nkv, old, BLOCK, size).float() * scale_k
    v8 = (state["values"][:, :old][..., _slots()].float() - 128.0).transpose(2, 3) * scale_v
    k8, v8 = k8.reshape(nkv, old * BLOCK, size), v8.reshape(nkv, old * BLOCK, size)
    k32, v32 = (_own_block_rows(state, w).transpose(0, 1) for w in range(2))
    group = nh // nkv
    q = state["q"].reshape(count, nkv, group, size).permute(1, 2, 0, 3).reshape(nkv, group * count, size)
    at = torch.arange(pos, pos + count, device="cuda").repeat(group)[:, None]
    block = at // BLOCK * BLOCK
    j8 = torch.arange(old * BLOCK, device="cuda")[None]
    j32 = torch.arange(first, first + k32.shape[1], device="cuda")[None]
    s8 = torch.matmul(q, k8.transpose(1, 2)).masked_fill_(~(j8 < block), -math.inf)
    s32 = torch.matmul(q, k32.transpose(1, 2)).masked_fill_(~((j32 >= block) & (j32 <= at)), -math.inf)
    s = torch.cat([s8, s32], -1).mul_(1.0 / math.sqrt(size))
    del s8, s32
    p = torch.exp(s.sub_(s.amax(-1, keepdim=True)))
    out = torch.matmul(p, torch.cat([v8, v32], 1)) / p.sum(-1, keepdim=True)
    return out.reshape(nkv, group, count, size).permute(2, 0, 1, 3).reshape(count, nh * size)


def _plain_logprobs(state):
    case = state["case"]
    x = state["logits"][:, :case["vocab"]]
    z = x - x.amax(-1, keepdim=True)
    e = torch.exp(z)
    total = e.sum(-1, keepdim=True)
    log_total = torch.log(total)
    entropy = (log_total - torch.where(e > 0, e * z, 0.0).sum(-1, keepdim=True) / total)[:, 0]
    logp = torch.gather(z, 1, state["given"].long()) - log_total
    if not case["top"]:
        return _outputs(logp, entropy, None, None, 0)
    best, at = torch.sort(z, dim=-1, descending=True, stable=True)
    best, at = best[:, :case["top"]], at[:, :case["top"]]
    return _outputs(logp, entropy, torch.where(torch.isinf(best), -1, at).to(torch.int32), best - log_total, case["top"])


# ---- what the call cannot do without


def work(case):
    if case["kind"] == "logprobs":
        values = case["rows"] * case["vocab"]
        small = case["rows"] * (4 * 2 * case["given"] + 4 + 8 * case["top"])
        return {"bytes": 4.0 * values + small, "flops": 6.0 * values}
    nh, nkv, size = HEADS[case["heads"]]
    pos, count, width = case["pos"], case["count"], nkv * size
    first = pos // BLOCK * BLOCK
    if case["kind"] == "append":
        whole = (pos + count) // BLOCK * BLOCK - first  # positions that become 8 bits
        whole = max(0, whole)
        eight = 2 * whole * width + whole // BLOCK * nkv * 8
        rows = 8 * count * width
        earlier = 8 * (pos - first) * width if whole else 0
        # rows in, 8 bits out (and the latest rows in float32), then 8 bits (or rows) in again and rows out
        return {"bytes": float(2 * rows + earlier + 2 * eight + 8 * min(count, RECENT) * width), "flops": 4.0 * count * width}
    old = (pos + count - 1) // BLOCK
    seen = sum(range(pos + 1, pos + count + 1))
    return {"bytes": float(old * (2 * BLOCK * width + 8 * nkv) + 8 * (pos - first + count) * width
                           + 8 * count * nh * size), "flops": 4.0 * nh * size * seen}


# ---- the same in 64 bits, from the definitions


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "logprobs":
        logp, entropy, ids, logps = [], [], [], []
        for x, given in zip(state["logits"], state["given"].long()):
            x = x[:case["vocab"]].double()
            p = torch.softmax(x, 0)
            lp = torch.log_softmax(x, 0)
            logp.append(lp[given])
            entropy.append(-torch.special.xlogy(p, p).sum())
            if case["top"]:
                # the largest, the lowest index first among equals
                order = sorted(((-v, i) for v, i in zip(*(t.tolist() for t in torch.topk(x, min(x.numel(), case["top"] + 8))))))
                ids.append(torch.tensor([i if v < math.inf else -1 for v, i in order[:case["top"]]], dtype=torch.int32))
                logps.append(torch.tensor([-v for v, i in order[:case["top"]]], dtype=torch.float64)
                             - torch.logsumexp(x, 0).item())
        return _outputs(torch.stack(logp), torch.stack(entropy), torch.stack(ids) if ids else None,
                        torch.stack(logps) if logps else None, case["top"])
    nh, nkv, size = HEADS[case["heads"]]
    pos, count = case["pos"], case["count"]
    first, end = pos // BLOCK * BLOCK, pos + count
    source = {}
    for which, name in enumerate(("keys", "values")):
        kept = state["recent_" + name].double()
        apart = case["kind"] == "attention" and end > first + RECENT
        rows = {p: kept[RECENT + p - first if apart else p % RECENT] for p in range(first, pos)}
        given = state["kv"[which]].double().reshape(count, nkv, size)
        source[name] = torch.cat([torch.stack([rows[p] for p in range(first, pos)]), given]) if rows else given
    if case["kind"] == "append":
        got = {}
        for name, rows in source.items():
            for b in range(0, end // BLOCK * BLOCK - first, BLOCK):
                for h in range(nkv):
                    x = rows[b:b + BLOCK, h]
                    s = (x.abs().max().float() / 127.0).double()
                    rows[b:b + BLOCK, h] = torch.round(x / s) * s if s > 0 else 0.0
            got[name] = rows[pos - first:].reshape(count, -1)
        return got
    if 4.0 * nh * size * count * end > 4e12:
        return None
    old = (end - 1) // BLOCK
    t = torch.arange(BLOCK, device="cuda")
    byte = 16 * (t // 4 % 2) + 8 * (t // 16) + 4 * (t // 8 % 2) + t % 4
    out = torch.empty(count, nh, size, dtype=torch.float64, device="cuda")
    q = state["q"].double().reshape(count, nh, size)
    for g in range(nkv):
        s = state["scales"][g, :old].double()
        # position 32 b + t, channel 16 c + i from [b][c][t][i]; from [b][channel][byte of t]
        k8 = (state["keys"][g, :old].double() * s[:, 0, None, None, None]).permute(0, 2, 1, 3).reshape(-1, size)
        v8 = ((state["values"][g, :old].double() - 128.0) * s[:, 1, None, None])[:, :, byte].permute(0, 2, 1)
        v8 = v8.reshape(-1, size)
        for a in range(0, count, 512):
            positions = torch.arange(pos + a, pos + min(count, a + 512), device="cuda")
            start = positions - positions % BLOCK
            lo = int(start[0])
            seen = int(start[-1])
            k = torch.cat([k8[:seen], source["keys"][lo - first:int(positions[-1]) + 1 - first, g]])
            v = torch.cat([v8[:seen], source["values"][lo - first:int(positions[-1]) + 1 - first, g]])
            j = torch.cat([torch.arange(seen, device="cuda"), torch.arange(lo, int(positions[-1]) + 1, device="cuda")])
            is8 = torch.arange(len(j), device="cuda") < seen
            visible = torch.where(is8[None], j[None] < start[:, None],
                                  (j[None] >= start[:, None]) & (j[None] <= positions[:, None]))
            for h in range(g * nh // nkv, (g + 1) * nh // nkv):
                score = q[a:a + 512, h] @ k.T / math.sqrt(size)
                out[a:a + 512, h] = torch.softmax(score.masked_fill(~visible, -math.inf), -1) @ v
    return out.reshape(count, nh * size)
