"""The operators over a cache in pages that several sequences share, and the products with 4-bit weights: what a program
gives hk_pages_fork, hk_pages_reserve, hk_pages_free, hk_pages_compact, hk_pages_append, hk_pages_attention and
hk_matmul_four. A case is a dict of plain values; `listed` names the fixed ones, `draw` makes more of the same ranges,
`prepare` is what a program holds before the call, `run` is the call (in its plain form by elementary torch operations, or
with `own` through the library), `work` its unavoidable bytes and operations, `exact` the same result from the definitions,
in 64 bits.

The cache: keys and values [layer][page][kv head][position][channel], float32 or float16. A sequence's row of the tables
names the page of each `page` positions (-1: none); refs counts the table entries that name a page (0: free).

The 4-bit matrices: w in -8..7 with a scale a row and `group` columns; 128 columns are 64 bytes, whose 16-byte chunk j
holds, in byte 4 t + i, column 32 t + 4 j + i (low four bits) and column 32 t + 16 + 4 j + i (high four bits). Rows are
filled up to a multiple of 128 columns with zeros.
"""
import ctypes
import importlib
import math

import numpy
import torch

own = False

# query heads, kv heads, head size and layers: the repository's own models and tests, and two generic layouts (wide heads,
# an odd group)
HEADS = {
    "llama3-8b": (32, 8, 128, 32),
    "qwen25-7b": (28, 4, 128, 28),
    "llm150m": (8, 8, 64, 12),
    "stories15m": (6, 6, 48, 6),
    "gpt2-small": (12, 12, 64, 12),
    "test-16": (4, 2, 16, 2),
    "test-96": (12, 4, 96, 2),
    "wide-256": (16, 8, 256, 4),
    "odd-32": (10, 5, 32, 3),
}
# rows and columns of the repository's own models' matrices
MATRICES = [(4096, 4096), (6144, 4096), (14336, 4096), (4096, 14336), (3584, 3584), (18944, 3584), (3584, 18944), (768, 768),
            (2304, 768), (288, 288), (768, 288), (288, 768), (32000, 288), (32000, 768), (128256, 4096), (152064, 3584)]
POOL = 1 << 30  # bytes of keys and values a case holds at most


def listed():
    return [
        # eight answers to each of two prompts begin: the last round's dropped, the prompts' pages shared, a page copied for
        # each answer's first token
        dict(name="branch-8b", kind="branch", heads="llama3-8b", half=True, page=64, parents=2, children=8, length=1000, grow=1),
        # four beams of the smallest model go on from one
        dict(name="branch-15m", kind="branch", heads="stories15m", half=False, page=32, parents=1, children=4, length=203, grow=1),
        # a pool that half of the conversations have left, before it is made smaller
        dict(name="compact-8b", kind="compact", heads="llama3-8b", half=True, page=64, pages=112, used=0.5, seqs=9),
        # many small pages
        dict(name="compact-150m", kind="compact", heads="llm150m", half=True, page=32, pages=900, used=0.8, seqs=40),
        # one token of each of 64 conversations into a layer
        dict(name="append-64", kind="append", heads="llama3-8b", half=True, page=64, rows=64, length=500, prompt=False),
        # a prompt's rows into a layer
        dict(name="append-prompt", kind="append", heads="llama3-8b", half=False, page=128, rows=2048, length=0, prompt=True),
        # the smallest model's step: launches and latency
        dict(name="token-15m", kind="attention", heads="stories15m", half=False, page=32, rows=1, longest=200, ragged=False, shared=0),
        # a step of 48 conversations of all lengths
        dict(name="step-48", kind="attention", heads="qwen25-7b", half=True, page=64, rows=48, longest=8000, ragged=True, shared=0),
        # two conversations over long documents
        dict(name="step-131k", kind="attention", heads="llama3-8b", half=True, page=64, rows=2, longest=131077, ragged=False, shared=0),
        # a decode step's product, one token
        dict(name="four-token", kind="four", rows=4096, k=4096, m=1, group=32, half=False, bias=64),
        # the classifier, one token: the most bytes
        dict(name="four-classifier", kind="four", rows=128256, k=4096, m=1, group=128, half=True, bias=64),
        # a decode step of 16 conversations
        dict(name="four-16", kind="four", rows=14336, k=4096, m=16, group=32, half=True, bias=64),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _row_bytes(case):
    """keys and values of one position of one layer"""
    _, nkv, size, _ = HEADS[case["heads"]]
    return 2 * nkv * size * (2 if case["half"] else 4)


def draw(rng):
    kind = rng.choice(["branch", "compact", "append", "attention", "attention", "four", "four"])
    if kind == "four":
        rows, k = rng.choice(MATRICES + [(_log_int(rng, 1, 20000), 32 * _log_int(rng, 1, 300))])
        m = _log_int(rng, 1, 64)
        while m > 1 and rows * k * m > 14336 * 4096 * 32:
            m //= 2
        return dict(kind=kind, rows=rows, k=k, m=m, group=rng.choice([32, 64, 128]), half=rng.random() < 0.5,
                    bias=rng.choice([0, 64]))
    case = dict(kind=kind, heads=rng.choice(sorted(HEADS)), half=rng.random() < 0.6, page=rng.choice([32, 64, 128]))
    each, layers = _row_bytes(case), HEADS[case["heads"]][3]
    if kind == "branch":
        case.update(parents=_log_int(rng, 1, 4), children=_log_int(rng, 1, 16), length=_log_int(rng, 1, 2000),
                    grow=rng.choice([1, 1, 1, 5, 70]))
        while _branch_pages(case) * case["page"] * each * layers > POOL // 2:
            case["length"], case["children"] = case["length"] * 2 // 3 + 1, case["children"] * 2 // 3 + 1
            case["parents"], case["grow"] = (case["parents"] + 1) // 2, min(case["grow"], 5)
        return case
    if kind == "compact":
        most = POOL // 2 // (case["page"] * each * layers)
        pages = _log_int(rng, min(8, most), min(2000, most))
        return dict(case, pages=pages, used=rng.choice([0.2, 0.5, 0.8, 0.95]), seqs=_log_int(rng, 1, min(64, pages)))
    if kind == "append":
        if rng.random() < 0.5:
            return dict(case, rows=_log_int(rng, 1, 128), length=_log_int(rng, 1, 1000) - 1, prompt=False)
        return dict(case, rows=_log_int(rng, 2, 2048), length=_log_int(rng, 1, 3000) - 1, prompt=True)
    rows = _log_int(rng, 1, 96)
    longest = _log_int(rng, 1, max(2, min(131077, POOL // each // rows)))
    shared = longest * rng.choice([0, 0, 1, 9]) // 10 // case["page"] * case["page"]
    return dict(case, rows=rows, longest=longest, ragged=rng.random() < 0.5, shared=shared)


# ---- what a program holds before the call


def _package():
    return importlib.import_module("pyodide-llm_amd")


def _generator(seed, stream):
    return torch.Generator(device="cuda").manual_seed((seed * 1000003 + stream) % (1 << 62))


def _randn(shape, seed, stream, dtype=torch.float32):
    return torch.randn(shape, device="cuda", generator=_generator(seed, stream), dtype=dtype)


def _order(n, seed, stream):
    return torch.randperm(n, device="cuda", generator=_generator(seed, stream)).to(torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _ceil(a, b):
    return -(-a // b)


def _branch_pages(case):
    """pages of a pool that a branch case fits in, and a few more"""
    own_pages = _ceil(case["length"] + case["grow"], case["page"]) - case["length"] // case["page"]
    return case["parents"] * (_ceil(case["length"], case["page"]) + case["children"] * own_pages) + 5


def _lengths(case):
    """the rows' lengths: all alike, or spread from one position to the longest"""
    n, longest = case["rows"], case["longest"]
    if not case["ragged"]:
        return [longest] * n
    return [1 + int((longest - 1) * ((i * 0.6180339887 + 0.999) % 1.0)) for i in range(n - 1)] + [longest]


def _pool(case, layers, pages, seed):
    _, nkv, size, _ = HEADS[case["heads"]]
    dtype = torch.float16 if case["half"] else torch.float32
    # keys with strong and weak channels, values around zero, as projections give them
    keys = _randn((layers, pages, nkv, case["page"], size), seed, 1, dtype)
    keys *= torch.exp(0.5 * _randn((nkv, 1, size), seed, 2)).to(dtype)
    return keys, _randn((layers, pages, nkv, case["page"], size), seed, 3, dtype)


def _counted(tables, pages):
    named = torch.where(tables < 0, pages, tables).long().flatten()
    return torch.zeros(pages + 1, dtype=torch.int64, device="cuda").index_add_(0, named, torch.ones_like(named))[:pages].to(torch.int32)


def _cache(case, keys, values, tables, **more):
    return dict(case=case, keys=keys, values=values, tables=tables, refs=_counted(tables, keys.shape[1]), handle=None, **more)


def _nibbles(w):
    """w int8 [rows][columns, a multiple of 128] -> bytes [rows][columns / 2]"""
    rows = w.shape[0]
    part = w.reshape(rows, -1, 4, 2, 4, 4).permute(3, 0, 1, 4, 2, 5)  # [low / high][row][of 128][j][t][i]
    return ((part[0] & 15) | (part[1] & 15) << 4).to(torch.uint8).reshape(rows, -1)


def _prepare_four(case, seed):
    rows, k, m, group = case["rows"], case["k"], case["m"], case["group"]
    wide = _ceil(k, 128) * 128
    w = torch.empty(rows, wide // 2, dtype=torch.uint8, device="cuda")
    ws = torch.empty(rows, wide // group, dtype=torch.float16 if case["half"] else torch.float32, device="cuda")
    for at in range(0, rows, 8192):  # a piece at a time: a large matrix is not held in float32
        n = min(8192, rows - at)
        x = torch.zeros(n, wide, device="cuda")
        x[:, :k] = 0.02 * _randn((n, k), seed, 10 + at)
        x = x.reshape(n, -1, group)
        s = (x.abs().amax(-1) / 7.0).to(ws.dtype)
        q = torch.where(s[..., None] > 0, torch.round(x / s[..., None].float()).clamp(-8, 7), 0.0)
        w[at:at + n] = _nibbles(q.to(torch.int8).reshape(n, wide))
        ws[at:at + n] = s
    # activations as quantize_x leaves them: a group of 32 by its largest magnitude, in 7 bits with 64 added or in 8
    x = _randn((m, k // 32, 32), seed, 1) * torch.exp(0.5 * _randn((1, k // 32, 32), seed, 2))
    most = 63.0 if case["bias"] else 127.0
    xs = x.abs().amax(-1) / most
    xq = torch.round(x / xs[..., None]).clamp(-most, most) + case["bias"]
    return dict(case=case, w=w, ws=ws, xq=xq.to(torch.int8).reshape(m, k), xs=xs, y=torch.empty(m, rows, device="cuda"))


def prepare(case, seed):
    if case["kind"] == "four":
        return _prepare_four(case, seed)
    nh, nkv, size, layers = HEADS[case["heads"]]
    page = case["page"]
    if case["kind"] == "branch":
        parents, children, length = case["parents"], case["children"], case["length"]
        pages, held = _branch_pages(case), _ceil(length, page)
        keys, values = _pool(case, layers, pages, seed)
        slots = _ceil(length + case["grow"], page) + 3
        tables = _ints([[-1] * slots] * (parents * (1 + children)))
        tables[:parents, :held] = _order(pages, seed, 4)[:parents * held].reshape(parents, held)
        n = parents * children
        return _cache(case, keys, values, tables, to=_ints(range(parents, parents + n)),
                      source=_ints([i // children for i in range(n)]), starts=_ints([length] * n),
                      ends=_ints([length + case["grow"]] * n), none=_ints([0] * n), status=_ints([0]))
    if case["kind"] == "compact":
        pages, seqs = case["pages"], case["seqs"]
        keys, values = _pool(case, layers, pages, seed)
        named = _order(pages, seed, 4)[:max(1, int(case["used"] * pages))]
        slots = _ceil(named.numel(), seqs) + 2
        tables = _ints([[-1] * slots] * seqs)
        at = torch.arange(named.numel(), device="cuda")
        tables[at % seqs, at // seqs] = named
        if seqs > 1:  # two conversations share a beginning
            tables[1, 0] = tables[0, 0]
        state = _cache(case, keys, values, tables, used=_ints([0]))
        state["before"] = (tables.clone(), state["refs"].clone())
        return state
    if case["kind"] == "append":
        rows, length = case["rows"], case["length"]
        seqs = 1 if case["prompt"] else rows
        ends = [length + rows] if case["prompt"] else [length + 1 + i % 7 for i in range(rows)]
        slots = max(_ceil(e, page) for e in ends) + 1
        pages = sum(_ceil(e, page) for e in ends) + 3
        keys, values = _pool(case, 1, pages, seed)
        tables, order, at = _ints([[-1] * slots] * seqs), _order(pages, seed, 4), 0
        for i, e in enumerate(ends):
            n = _ceil(e, page)
            tables[i, :n] = order[at:at + n]
            at += n
        positions = range(length, length + rows) if case["prompt"] else [e - 1 for e in ends]
        return _cache(case, keys, values, tables, k=_randn((rows, nkv * size), seed, 5), v=_randn((rows, nkv * size), seed, 6),
                      seqs=_ints([0] * rows if case["prompt"] else range(rows)), positions=_ints(list(positions)))
    rows, lengths, common = case["rows"], _lengths(case), case["shared"] // page
    held = [max(0, _ceil(n, page) - common) for n in lengths]
    pages = common + sum(held) + 2
    keys, values = _pool(case, 1, pages, seed)
    tables, order, at = _ints([[-1] * (_ceil(case["longest"], page) + 1)] * rows), _order(pages, seed, 4), common
    for i, n in enumerate(held):
        both = min(common, _ceil(lengths[i], page))
        tables[i, :both] = order[:both]
        tables[i, common:common + n] = order[at:at + n]
        at += n
    q = 1.5 * _randn((rows, nh * size), seed, 5)
    # (a step's conversations come in any order)
    seqs = _order(rows, seed, 6)
    return _cache(case, keys, values, tables, q=q, out=torch.empty_like(q), seqs=seqs, lengths=_ints(lengths)[seqs.long()])


# ---- the call


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"branch": _own_branch, "compact": _own_compact, "append": _own_append, "attention": _own_attention,
                "four": _own_four}[kind](state)
    return {"branch": _plain_branch, "compact": _plain_compact, "append": _plain_append, "attention": _plain_attention,
            "four": _plain_four}[kind](state)


def _handle(state):
    """the hk_pages over the state's buffers and a workspace, made once, as a program keeps them"""
    if state["handle"] is None:
        pk, case, keys = _package(), state["case"], state["keys"]
        nh, nkv, size, _ = HEADS[case["heads"]]
        pages = pk.HkPages(keys=keys.data_ptr(), values=state["values"].data_ptr(), tables=state["tables"].data_ptr(),
                           refs=state["refs"].data_ptr(), n_layers=keys.shape[0], n_pages=keys.shape[1], n_kv_heads=nkv,
                           page_size=case["page"], head_size=size, half=int(case["half"]), n_seqs=state["tables"].shape[0],
                           table_size=state["tables"].shape[1])
        if case["kind"] == "attention":
            need = pk.library().hk_pages_attention_workspace(ctypes.byref(pages), nh, case["rows"], case["longest"])
        else:
            need = pk.library().hk_pages_workspace(ctypes.byref(pages))
        space = torch.empty(max(1, need), dtype=torch.uint8, device="cuda")
        if case["kind"] == "branch":  # (a fork's status beside the reserve's: each call writes its own)
            state["forked"] = torch.zeros_like(state["status"])
        state["handle"] = (pk.library(), pk.hip_engine.check, ctypes.byref(pages), space, need)
    return state["handle"]


def _own_branch(state):
    lib, check, pages, space, need = _handle(state)
    stream, n, to = torch.cuda.current_stream().cuda_stream, state["to"].numel(), state["to"].data_ptr()
    starts, status = state["starts"].data_ptr(), state["status"].data_ptr()
    check(lib.hk_pages_free(pages, to, state["none"].data_ptr(), n, stream))
    check(lib.hk_pages_fork(pages, to, state["source"].data_ptr(), starts, n, state["forked"].data_ptr(), stream))
    check(lib.hk_pages_reserve(pages, to, starts, state["ends"].data_ptr(), n, status, space.data_ptr(), need, stream))
    return {name: state[name] for name in ("tables", "refs", "status", "keys", "values")}


def _own_compact(state):
    lib, check, pages, space, need = _handle(state)
    for now, before in zip((state["tables"], state["refs"]), state["before"]):
        now.copy_(before)
    check(lib.hk_pages_compact(pages, state["used"].data_ptr(), space.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    return {name: state[name] for name in ("tables", "refs", "used", "keys", "values")}


def _own_append(state):
    lib, check, pages, _, _ = _handle(state)
    k = state["k"]
    check(lib.hk_pages_append(pages, 0, k.data_ptr(), state["v"].data_ptr(), k.shape[1], state["seqs"].data_ptr(),
                              state["positions"].data_ptr(), k.shape[0], torch.cuda.current_stream().cuda_stream))
    return {"keys": state["keys"], "values": state["values"]}


def _own_attention(state):
    lib, check, pages, space, need = _handle(state)
    case, out, width = state["case"], state["out"], state["q"].shape[1]
    check(lib.hk_pages_attention(out.data_ptr(), state["q"].data_ptr(), pages, 0, HEADS[case["heads"]][0], width, width,
                                 state["seqs"].data_ptr(), state["lengths"].data_ptr(), case["rows"], case["longest"],
                                 space.data_ptr(), need, torch.cuda.current_stream().cuda_stream))
    return out


def _own_four(state):
    pk, case, y = _package(), state["case"], state["y"]
    pk.hip_engine.check(pk.library().hk_matmul_four(
        y.data_ptr(), state["xq"].data_ptr(), state["xs"].data_ptr(), state["w"].data_ptr(), state["ws"].data_ptr(), case["m"],
        case["rows"], case["k"], case["bias"], case["group"], int(case["half"]), torch.cuda.current_stream().cuda_stream))
    return y


def _plain_count(state, entries, by):
    """refs + by for every page that entries name"""
    refs = torch.cat([state["refs"], state["refs"].new_zeros(1)])
    named = torch.where(entries < 0, refs.numel() - 1, entries).long().flatten()
    refs.index_add_(0, named, torch.full_like(named, by, dtype=torch.int32))
    state["refs"].copy_(refs[:-1])


def _plain_branch(state):
    tables, refs, page = state["tables"], state["refs"], state["case"]["page"]
    to, source = state["to"].long(), state["source"].long()
    slot = torch.arange(tables.shape[1], device="cuda")[None]
    # the last round's
    _plain_count(state, tables[to], -1)
    tables[to] = -1
    # the parents' pages
    begun = torch.where(slot * page < state["starts"][:, None], tables[source], -1)
    _plain_count(state, begun, 1)
    # room for what comes: the lowest free pages where there is none yet, or one that others read
    written = (slot >= (state["starts"] // page)[:, None]) & (slot * page < state["ends"][:, None])
    new = written & ((begun < 0) | (refs[begun.clamp(min=0).long()] > 1))
    free = torch.sort((refs > 0).to(torch.int32), stable=True)[1]
    taken = free[(torch.cumsum(new.flatten(), 0) - 1).clamp(min=0)].reshape(new.shape).to(torch.int32)
    lacking = (new.sum() - (refs == 0).sum()).clamp(min=0)
    after = torch.where(new, taken, begun)
    _plain_count(state, torch.where(new, begun, -1), -1)
    _plain_count(state, torch.where(new, taken, -1), 1)
    tables[to] = after
    # the rows before the first written one
    at = (state["starts"] // page).long()[:, None]
    old, own_page = torch.gather(begun, 1, at)[:, 0], torch.gather(after, 1, at)[:, 0].long()
    kept = torch.arange(page, device="cuda")[None] < (state["starts"] % page)[:, None]
    kept = (kept & (old >= 0)[:, None])[None, :, None, :, None]
    for pool in (state["keys"], state["values"]):
        pool[:, own_page] = torch.where(kept, pool[:, old.clamp(min=0).long()], pool[:, own_page])
    state["status"].copy_(lacking[None])
    return {name: state[name] for name in ("tables", "refs", "status", "keys", "values")}


def _plain_compact(state):
    for now, before in zip((state["tables"], state["refs"]), state["before"]):
        now.copy_(before)
    refs, tables = state["refs"], state["tables"]
    at = torch.arange(refs.numel(), device="cuda")
    used = (refs > 0).sum()
    holes, moved = ((refs == 0) & (at < used)).nonzero()[:, 0], ((refs > 0) & (at >= used)).nonzero()[:, 0]
    place = at.to(torch.int32)
    place[moved] = holes.to(torch.int32)
    for pool in (state["keys"], state["values"]):
        pool[:, holes] = pool[:, moved]
    refs[holes] = refs[moved]
    refs[moved] = 0
    tables.copy_(torch.where(tables < 0, tables, place[tables.clamp(min=0).long()]))
    state["used"].copy_(used[None])
    return {name: state[name] for name in ("tables", "refs", "used", "keys", "values")}


def _plain_append(state):
    keys, page = state["keys"], state["case"]["page"]
    nkv, size = keys.shape[2], keys.shape[4]
    positions = state["positions"].long()
    held = state["tables"][state["seqs"].long(), positions // page].long()
    for pool, rows in ((keys, state["k"]), (state["values"], state["v"])):
        pool[0, held, :, positions % page] = rows.reshape(-1, nkv, size).to(pool.dtype)
    return {"keys": keys, "values": state["values"]}


def _plain_attention(state):
    case = state["case"]
    nh, nkv, size, _ = HEADS[case["heads"]]
    rows, page = case["rows"], case["page"]
    out = torch.empty_like(state["q"])
    q = state["q"].reshape(rows, nkv, nh // nkv, size)
    slots = _ceil(case["longest"], page)
    at = torch.arange(slots * page, device="cuda")
    step = max(1, 48 * 8000 // (slots * page))  # (rows at a time, so that a long step's float32 rows fit)
    for a in range(0, rows, step):
        held = state["tables"][state["seqs"][a:a + step].long(), :slots].clamp(min=0).long()
        n = held.shape[0]
        k, v = (pool[0, held].float().permute(0, 2, 1, 3, 4).reshape(n, nkv, slots * page, size)
                for pool in (state["keys"], state["values"]))
        seen = (at[None] < state["lengths"][a:a + step, None])[:, None, None]
        s = torch.matmul(q[a:a + step], k.transpose(2, 3)) * (1.0 / math.sqrt(size))
        s = torch.where(seen, s, -math.inf)
        p = torch.exp(s - s.amax(-1, keepdim=True))
        v = torch.where(seen[:, 0, 0, :, None][:, None], v, 0.0)
        out[a:a + step] = (torch.matmul(p, v) / p.sum(-1, keepdim=True)).reshape(n, nh * size)
    return out


def _columns(w):
    """bytes [rows][columns / 2] -> int8 [rows][columns]"""
    part = w.reshape(w.shape[0], -1, 4, 4, 4)  # [row][of 128][j][t][i]
    both = torch.stack([part & 15, part >> 4], 2).to(torch.int8)  # [row][of 128][low / high][j][t][i]
    both = both.permute(0, 1, 4, 2, 3, 5).reshape(w.shape[0], -1)
    return torch.where(both > 7, both - 16, both)


def _plain_four(state):
    case = state["case"]
    rows, k, m = case["rows"], case["k"], case["m"]
    x = ((state["xq"].float() - case["bias"]).reshape(m, k // 32, 32) * state["xs"][..., None]).reshape(m, k)
    y = torch.empty(m, rows, device="cuda")
    for at in range(0, rows, 32768):
        w = _columns(state["w"][at:at + 32768]).float().reshape(-1, state["ws"].shape[1], case["group"])
        w = (w * state["ws"][at:at + 32768, :, None].float()).reshape(w.shape[0], -1)[:, :k]
        y[:, at:at + 32768] = torch.matmul(x, w.transpose(0, 1))
    return y


# ---- what the call cannot do without


def work(case):
    if case["kind"] == "four":
        rows, k, m = case["rows"], case["k"], case["m"]
        weights = rows * (k / 2 + _ceil(k, case["group"]) * (2 if case["half"] else 4))
        return {"bytes": float(weights + m * (k + k / 8 + 4 * rows)), "flops": 2.0 * m * rows * k}
    nh, nkv, size, layers = HEADS[case["heads"]]
    page, each = case["page"], _row_bytes(case)
    if case["kind"] == "branch":
        n, slots = case["parents"] * case["children"], _ceil(case["length"] + case["grow"], page)
        copied = n * (case["length"] % page) * each * layers
        # the rows copied, the parents' entries read and the children's written, the counts
        return {"bytes": float(2 * copied + 4 * (case["parents"] + n) * slots + 4 * _branch_pages(case)), "flops": float(n * slots)}
    if case["kind"] == "compact":
        pages = case["pages"]
        used = max(1, int(case["used"] * pages))
        # (the used pages lie anywhere: as many of them as lie past the used count, on average)
        moved = used * (pages - used) / pages
        slots = case["seqs"] * (_ceil(used, case["seqs"]) + 2)
        return {"bytes": float(2 * moved * page * each * layers + 8 * slots + 8 * pages), "flops": float(pages)}
    if case["kind"] == "append":
        return {"bytes": float(case["rows"] * (8 * nkv * size + each + 8)), "flops": float(2 * case["rows"] * nkv * size)}
    lengths, shared = _lengths(case), case["shared"]
    seen = sum(lengths)
    held = sum(max(0, n - shared) for n in lengths) + min(shared, max(lengths))
    return {"bytes": float(held * each + 8 * case["rows"] * nh * size), "flops": 4.0 * nh * size * seen}


# ---- the same from the definitions, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "four":
        return _exact_four(state)
    if case["kind"] == "attention":
        return _exact_attention(state)
    keys, values = state["keys"], state["values"]
    page = case["page"]
    tables, refs = state["tables"].cpu().numpy(), state["refs"].cpu().numpy()
    if case["kind"] == "append":
        nkv, size = keys.shape[2], keys.shape[4]
        got = {"keys": keys.double(), "values": values.double()}
        for name, rows in (("keys", state["k"]), ("values", state["v"])):
            rows = rows.double().reshape(-1, nkv, size)
            for i, (s, p) in enumerate(zip(state["seqs"].tolist(), state["positions"].tolist())):
                got[name][0, int(tables[s, p // page]), :, p % page] = rows[i]
        return got
    if case["kind"] == "compact":
        used = int((refs > 0).sum())
        free = [p for p in range(used) if refs[p] == 0]
        for new, old in zip(free, [p for p in range(used, len(refs)) if refs[p] > 0]):
            keys[:, new], values[:, new] = keys[:, old], values[:, old]
            refs[new], refs[old] = refs[old], 0
            tables[tables == old] = new
        return {"tables": torch.from_numpy(tables), "refs": torch.from_numpy(refs), "used": _ints([used]), "keys": keys,
                "values": values}
    length, end = case["length"], case["length"] + case["grow"]
    for child, parent in zip(state["to"].tolist(), state["source"].tolist()):
        for j in range(_ceil(length, page)):
            tables[child, j] = tables[parent, j]
            refs[tables[child, j]] += 1
    before = refs.copy()
    free = iter([p for p in range(len(refs)) if refs[p] == 0])
    for child in state["to"].tolist():
        for j in range(length // page, _ceil(end, page)):
            old = tables[child, j]
            if old >= 0 and before[old] <= 1:
                continue
            new = next(free)
            if old >= 0:
                refs[old] -= 1
                kept = length - j * page
                keys[:, new, :, :kept], values[:, new, :, :kept] = keys[:, old, :, :kept], values[:, old, :, :kept]
            tables[child, j], refs[new] = new, 1
    return {"tables": torch.from_numpy(tables), "refs": torch.from_numpy(refs), "status": _ints([0]), "keys": keys,
            "values": values}


def _exact_attention(state):
    case = state["case"]
    nh, nkv, size, _ = HEADS[case["heads"]]
    page, group = case["page"], nh // nkv
    out = torch.empty(case["rows"], nh, size, dtype=torch.float64, device="cuda")
    q = state["q"].double().reshape(case["rows"], nh, size)
    tables = state["tables"].cpu()
    for i, (s, n) in enumerate(zip(state["seqs"].tolist(), state["lengths"].tolist())):
        held = tables[s, :_ceil(n, page)].to("cuda", torch.int64)
        for g in range(nkv):
            k, v = (pool[0, held, g].reshape(-1, size)[:n].double() for pool in (state["keys"], state["values"]))
            p = torch.softmax((k @ q[i, g * group:(g + 1) * group].T) / math.sqrt(size), 0)
            out[i, g * group:(g + 1) * group] = p.T @ v
    return out.reshape(case["rows"], nh * size)


def _exact_four(state):
    case = state["case"]
    rows, k, m = case["rows"], case["k"], case["m"]
    x = (state["xq"].double() - case["bias"]) * state["xs"].double().repeat_interleave(32, 1)
    # where each column's four bits lie, one column at a time
    column = numpy.arange(k)
    of, t, high, j, i = column // 128, column // 32 % 4, column // 16 % 2, column // 4 % 4, column % 4
    byte, shift = torch.from_numpy(64 * of + 16 * j + 4 * t + i).cuda(), torch.from_numpy(4 * high).cuda()
    y = torch.empty(m, rows, dtype=torch.float64, device="cuda")
    for at in range(0, rows, 8192):
        four = state["w"][at:at + 8192].long()[:, byte] >> shift & 15
        w = (four - 16 * (four >> 3)).double() * state["ws"][at:at + 8192].double().repeat_interleave(case["group"], 1)[:, :k]
        y[:, at:at + 8192] = x @ w.T
    return y
