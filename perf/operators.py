"""Cases for the serving operators that surround paged decode attention.

Three operators of one token step over the paged KV cache, each in its plain
form (elementary torch operations, `own` false) and as the call a program
makes of this library (`own` true):

* append    - kk_kv_append_rope: a ragged batch of token rows, keys and
              queries rotated to their positions, keys and values written into
              the micro / extent pages;
* attention - kk_prefix_attention: decode attention of lanes that share a long
              prefix, whose pages are read once for all of them;
* logits    - kk_logits_process: repetition, presence and frequency
              penalties, biases and grammar masks on the logits, and the
              greedy token.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

NONE = 0xFFFFFFFF


# ---- cases ------------------------------------------------------------------


def listed():
    def append(name, rows, seqs, padded, q_heads, kv_heads, head_dim, rotary, page, far):
        return {"name": name, "op": "append", "rows": rows, "seqs": seqs, "padded": padded, "q_heads": q_heads,
                "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rotary, "page": page, "far": far}

    def attention(name, groups, lanes, prefix, suffix, q_heads, kv_heads, page, chunk):
        return {"name": name, "op": "attention", "groups": groups, "lanes": lanes, "prefix": prefix,
                "suffix": suffix, "q_heads": q_heads, "kv_heads": kv_heads, "page": page, "chunk": chunk}

    def logits(name, rows, vocab, history, bias, masked, penalties):
        return {"name": name, "op": "logits", "rows": rows, "vocab": vocab, "history": history, "bias": bias,
                "masked": masked, "penalties": penalties}

    return [
        # One new token of one request, the model shape of the benchmark: launch latency.
        append("append one token", 1, 1, 0, 32, 4, 64, 64, 8, 2048),
        # A decode batch of 64 lanes, five of its rows padding, at positions up to 4096.
        append("append decode batch", 64, 59, 5, 32, 4, 64, 64, 8, 4096),
        # A ragged prefill of odd length into a 16-token fixed-page pool, half of each head rotated.
        append("append ragged prefill", 4999, 7, 37, 16, 2, 128, 64, 16, 100000),
        # A large prefill batch at far positions of a long-context model.
        append("append large prefill", 16384, 24, 0, 32, 8, 128, 128, 8, 1000000),
        # Four requests forked from one short prompt: launch latency.
        attention("prefix few lanes", 1, 4, 259, 24, 32, 4, 8, False),
        # A decode batch with one system prompt and ragged conversations behind it.
        attention("prefix decode batch", 1, 32, 2048, 1024, 32, 4, 8, False),
        # A 64-position chunk of a long prompt: every position sees what stands before the chunk.
        attention("prefix prompt chunk", 1, 64, 8143, 64, 32, 4, 16, True),
        # Many samples of two long documents, one KV head for every eight query heads.
        attention("prefix long documents", 2, 64, 32749, 200, 32, 4, 8, False),
        # One lane with short history: launch latency.
        logits("logits one lane", 1, 32000, 200, 4, False, True),
        # The decode batch of the benchmark with grammar masks on some lanes.
        logits("logits decode batch", 32, 32000, 4096, 64, True, True),
        # An odd vocabulary (rows that start anywhere), masks and biases alone.
        logits("logits odd vocabulary", 61, 50021, 0, 300, True, False),
        # A large batch over a large vocabulary with long histories.
        logits("logits large batch", 256, 128000, 16384, 300, True, True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["append", "attention", "logits"])
    if op == "append":
        rows = _log(rng, 1, 16384)
        kv_heads = rng.choice([1, 2, 4, 8])
        head_dim = rng.choice([64, 128])
        return {"op": op, "rows": rows, "seqs": _log(rng, 1, min(rows, 64)), "padded": rng.randint(0, rows // 10),
                "q_heads": kv_heads * rng.choice([1, 2, 4] if kv_heads == 8 else [1, 3, 4, 7, 8]),
                "kv_heads": kv_heads, "head_dim": head_dim, "rotary": rng.choice([head_dim, head_dim // 2]),
                "page": rng.choice([8, 16, 32, 64]), "far": _log(rng, 2048, 1000000) + 16384}
    if op == "attention":
        kv_heads = rng.choice([1, 2, 4, 8])
        ratio = rng.choice([1, 3, 4, 7, 8] if kv_heads < 8 else [1, 2, 4])
        groups = rng.choice([1, 1, 2, 3])
        lanes = _log(rng, 2, 64 if groups <= 2 else 42)
        most = min(32749, 32749 * 4096 // (groups * lanes * kv_heads * ratio))
        return {"op": op, "groups": groups, "lanes": lanes, "prefix": _log(rng, 100, most),
                "suffix": _log(rng, 1, 1024), "q_heads": kv_heads * ratio, "kv_heads": kv_heads,
                "page": rng.choice([8, 8, 16, 32, 64]), "chunk": rng.random() < 0.25}
    rows = _log(rng, 1, 256)
    vocab = _log(rng, 1000, 128000)
    return {"op": op, "rows": rows, "vocab": vocab, "history": _log(rng, 1, 16384), "bias": rng.choice([0, 5, 300]),
            "masked": rng.random() < 0.6, "penalties": rng.random() < 0.8}


# ---- inputs -----------------------------------------------------------------


def _package():
    if "kim_kvcache_b200" not in sys.modules:
        path = os.path.join(os.getcwd(), "kim-kvcache_b200", "__init__.py")
        spec = importlib.util.spec_from_file_location("kim_kvcache_b200", path)
        module = importlib.util.module_from_spec(spec)
        sys.modules["kim_kvcache_b200"] = module
        spec.loader.exec_module(module)
    return sys.modules["kim_kvcache_b200"]


def _up(array):
    return torch.from_numpy(np.ascontiguousarray(array)).cuda()


class _Pages:
    """Hands out random distinct page slots of a micro and an extent pool."""

    def __init__(self, rng, micro, extent):
        self.micro, self.extent = rng.permutation(max(micro, 1)), rng.permutation(max(extent, 1))
        self.used = [0, 0]

    def take(self, kind, n):
        pool = self.extent if kind else self.micro
        got = pool[self.used[kind]:self.used[kind] + n]
        self.used[kind] += n
        return got


def _pools(state, c, layers, micro, extent, gen):
    """Both pools in one allocation of token rows, and one spare row behind them."""
    row = c["kv_heads"] * state["head_dim"]
    n_micro, n_extent = micro * layers * 2 * c["page"], extent * layers * 2 * 64
    storage = torch.randn(n_micro + n_extent + 1, row, generator=gen, device="cuda", dtype=torch.float16)
    state.update(storage=storage, layers=layers, micro=micro, extent=extent, n_micro=n_micro, row=row)


def _flat_rows(state, c, kind, slot, token, component):
    """Row of `storage` that holds (kind, slot, token) of the state's layer."""
    cap = np.where(kind == 1, 64, c["page"])
    at = ((slot.astype(np.int64) * state["layers"] + state["layer"]) * 2 + component) * cap + token
    return np.where(kind == 1, state["n_micro"] + at, at)


def prepare(case, seed):
    c = case
    rng = np.random.RandomState(seed % (1 << 31))
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"append": _prepare_append, "attention": _prepare_attention, "logits": _prepare_logits}[c["op"]](c, rng, gen)


def _prepare_append(c, rng, gen):
    s = {"case": c, "head_dim": c["head_dim"], "layer": 1}
    rows, live = c["rows"], c["rows"] - c["padded"]
    seqs = min(c["seqs"], live)
    cuts = np.sort(rng.choice(np.arange(1, live), seqs - 1, replace=False)) if seqs > 1 else np.zeros(0, int)
    lens = np.diff(np.concatenate([[0], cuts, [live]]))
    # Sequence by sequence: consecutive positions; whole runs of 64 tokens stand in extents or in small pages.
    position, run = np.zeros(live, np.int64), np.zeros(live, np.int64)
    at, runs = 0, 0
    for n in lens:
        first = rng.randint(0, c["far"] - int(n))
        position[at:at + n] = first + np.arange(n)
        run[at:at + n] = runs + position[at:at + n] // 64 - first // 64
        runs = run[at + n - 1] + 1
        at += n
    small, most = 64 // c["page"], live // 64 + 2 * seqs
    extents = int(0.7 * most) if c["page"] == 8 else 0
    run_kind = rng.permutation((np.arange(most) < extents).astype(np.int64))[:runs]
    pages = _Pages(rng, (most - extents) * small, extents)
    run_slots = np.zeros((runs, small), np.int64)
    run_slots[run_kind == 1, 0] = pages.take(1, int(run_kind.sum()))
    run_slots[run_kind == 0] = pages.take(0, int((run_kind == 0).sum()) * small).reshape(-1, small)
    kind = run_kind[run]
    offset = position % 64
    slot = np.where(kind == 1, run_slots[run, 0], run_slots[run, offset // c["page"]])
    token = np.where(kind == 1, offset, offset % c["page"])
    _pools(s, c, 2, (most - extents) * small, extents, gen)
    # Padding rows stand behind the last sequence.
    slots = np.zeros((rows, 2), np.int32)
    slots[:live, 0] = slot
    slots[:live, 1] = token | (kind << 16) | (1 << 24)
    positions = np.zeros(rows, np.int32)
    positions[:live] = position
    width = (c["q_heads"] + 2 * c["kv_heads"]) * c["head_dim"]
    s["qkv"] = torch.randn(rows, width, generator=gen, device="cuda").half()
    s["q_out"] = torch.randn(rows, c["q_heads"] * c["head_dim"], generator=gen, device="cuda").half()
    s.update(slots=_up(slots), positions=_up(positions), host_slots=slots, host_positions=positions)
    if own:
        kk = _package()
        s["call"], s["kk"] = kk.kernels()["kv_append_rope"], kk
        d = kk.KvAppendDesc()
        d.pools = _kk_pools(kk, s, c)
        d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = s["layer"], rows, c["q_heads"], c["rotary"], 10000.0
        d.slots, d.positions = s["slots"].data_ptr(), s["positions"].data_ptr()
        q_width, k_width = c["q_heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        base = s["qkv"].data_ptr()
        d.query, d.key, d.value = base, base + 2 * q_width, base + 2 * (q_width + k_width)
        d.query_stride = d.key_stride = d.value_stride = width
        d.query_out, d.query_out_stride = s["q_out"].data_ptr(), q_width
        s["desc"] = d
    return s


def _kk_pools(kk, s, c):
    base = s["storage"].data_ptr()
    return kk.KvPools(base, base + 2 * int(s["n_micro"]) * s["row"] if s["extent"] else 0, int(s["micro"]),
                      int(s["extent"]), s["layers"], c["kv_heads"], s["head_dim"], c["page"])


def _table(tokens, page, pages):
    """[n, 4] page descriptors (slot, first token, valid tokens, kind) of a sequence of `tokens` tokens."""
    full = tokens // 64 if page == 8 else 0
    small = -(-(tokens - 64 * full) // page)
    t = np.zeros((full + small, 4), np.int64)
    t[:full, 0], t[:full, 1], t[:full, 2], t[:full, 3] = pages.take(1, full), np.arange(full) * 64, 64, 1
    t[full:, 0], t[full:, 1], t[full:, 2] = pages.take(0, small), 64 * full + np.arange(small) * page, page
    if small:
        t[-1, 2] = tokens - t[-1, 1]
    return t


def _token_rows(s, c, table, component):
    """Row of `storage` of every token of a table, in order."""
    slot, kind = np.repeat(table[:, 0], table[:, 2]), np.repeat(table[:, 3], table[:, 2])
    token = np.arange(int(table[:, 2].sum())) - np.repeat(table[:, 1] - table[0, 1], table[:, 2]) if len(table) else np.zeros(0, int)
    return _flat_rows(s, c, kind, slot, token, component)


def _prepare_attention(c, rng, gen):
    s = {"case": c, "head_dim": 64, "layer": 1}
    groups, lanes, prefix = c["groups"], c["lanes"], c["prefix"]
    if c["chunk"]:  # positions of one chunk per group: lane i sees its first i + 1 tokens
        own_tokens = np.tile(np.arange(1, lanes + 1), groups)
    else:  # ragged; some lanes have nothing of their own yet
        own_tokens = rng.randint(0, c["suffix"] + 1, groups * lanes)
        own_tokens[0], own_tokens[-1] = 0, c["suffix"]
    sizes = [prefix] * groups + ([lanes] * groups if c["chunk"] else list(own_tokens))
    full = [n // 64 if c["page"] == 8 else 0 for n in sizes]
    micro = sum(-(-(n - 64 * f) // c["page"]) for n, f in zip(sizes, full))
    pages = _Pages(rng, micro, sum(full))
    _pools(s, c, 2, micro + 1, sum(full), gen)
    shared = [_table(prefix, c["page"], pages) for _ in range(groups)]
    if c["chunk"]:
        chunks = [_table(lanes, c["page"], pages) for _ in range(groups)]
        tails = []
        for b, n in enumerate(own_tokens):
            t = chunks[b // lanes]
            t = t[t[:, 1] < n].copy()
            t[-1, 2] = n - t[-1, 1]
            tails.append(t)
    else:
        tails = [_table(int(n), c["page"], pages) for n in own_tokens]
    most = max(1, int(own_tokens.max()))
    # The plain form's index of the same tables: rows of K of every token, and which of the padded ones count.
    s["prefix_k"] = _up(np.stack([_token_rows(s, c, t, 0) for t in shared]))
    s["prefix_v"] = _up(np.stack([_token_rows(s, c, t, 1) for t in shared]))
    tail = np.full((2, groups * lanes, most), len(s["storage"]) - 1, np.int64)
    for b, t in enumerate(tails):
        for component in (0, 1):
            r = _token_rows(s, c, t, component)
            tail[component, b, :len(r)] = r
    s["tail_k"], s["tail_v"], s["tail_n"] = _up(tail[0]), _up(tail[1]), _up(own_tokens)
    # Each lane's block table as the runtime has it: the shared pages, then its own.
    tables = []
    for b, t in enumerate(tails):
        t = t.copy()
        t[:, 1] += prefix
        tables.append(np.concatenate([shared[b // lanes], t]))
    s.update(tables=tables, scale=0.125)
    s["query"] = (torch.randn(groups * lanes, c["q_heads"] * 64, generator=gen, device="cuda") * 1.5).half()
    if own:
        kk = _package()
        k = kk.kernels()
        n_lanes = groups * lanes
        descs = (kk.PageDesc * sum(map(len, tables)))()
        flat = np.concatenate(tables)
        raw = np.zeros((len(flat), 4), np.uint32)
        raw[:, 0], raw[:, 1], raw[:, 2] = flat[:, 0], flat[:, 1], flat[:, 2] | (flat[:, 3] << 16)
        ctypes.memmove(descs, raw.ctypes.data, raw.nbytes)
        lane_array = (kk.AttnLane * n_lanes)()
        at = 0
        for b, t in enumerate(tables):
            lane_array[b].desc_offset, lane_array[b].desc_count = at, len(t)
            lane_array[b].token_count, lane_array[b].query_row = int(t[:, 2].sum()), b
            at += len(t)
        group_array = (kk.PrefixGroup * n_lanes)()
        n_groups = k["prefix_groups"](descs, lane_array, n_lanes, 2, 64, group_array, n_lanes)
        items, plan = (kk.PrefixItem * 65536)(), kk.PrefixPlan()
        rc = k["prefix_attention_plan"](descs, len(flat), lane_array, n_lanes, group_array, n_groups, c["q_heads"],
                                        c["kv_heads"], 148, items, 65536, ctypes.byref(plan))
        if rc != 0 or plan.num_items > 65536:
            raise RuntimeError("kk_prefix_attention_plan: %d" % rc)

        def device(array, count):
            return _up(np.frombuffer(array, np.uint8, max(1, count) * ctypes.sizeof(array._type_)).copy())

        s["plan"] = [device(descs, len(flat)), device(lane_array, n_lanes), device(group_array, n_groups),
                     device(items, plan.num_items)]
        size = k["prefix_attention_workspace_bytes"](ctypes.byref(plan))
        s["workspace"] = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        s["output"] = torch.empty_like(s["query"])
        d = kk.PrefixAttnDesc()
        d.pools, d.layer, d.q_heads, d.scale, d.plan = _kk_pools(kk, s, c), s["layer"], c["q_heads"], s["scale"], plan
        d.descs, d.lanes, d.groups, d.items = (t.data_ptr() for t in s["plan"])
        d.query, d.query_stride = s["query"].data_ptr(), c["q_heads"] * 64
        d.output, d.output_stride = s["output"].data_ptr(), c["q_heads"] * 64
        d.workspace, d.workspace_bytes = s["workspace"].data_ptr(), size
        s.update(desc=d, call=k["prefix_attention"], kk=kk)
    return s


def _prepare_logits(c, rng, gen):
    s = {"case": c}
    rows, vocab = c["rows"], c["vocab"]
    s["logits"] = torch.randn(rows, vocab, generator=gen, device="cuda") * 3.0
    if c["penalties"]:
        lens = rng.randint(c["history"] // 4, c["history"] + 1, rows)
        offsets = np.concatenate([[0], np.cumsum(lens)])
        # Text repeats itself: half of the tokens come from the vocabulary's first part.
        text = np.where(rng.rand(offsets[-1]) < 0.5, rng.randint(0, max(1, vocab // 50), offsets[-1]),
                        rng.randint(0, vocab, offsets[-1]))
        s["history"], s["history_offsets"] = _up(text.astype(np.int32)), _up(offsets.astype(np.int32))
        s["prompt_counts"] = _up((lens * rng.rand(rows)).astype(np.int32))
        some = rng.rand(3, rows) < 0.75
        s["repetition"] = _up(np.where(some[0], rng.uniform(1.0, 1.5, rows), 1.0).astype(np.float32))
        s["presence"] = _up(np.where(some[1], rng.uniform(-0.5, 1.0, rows), 0.0).astype(np.float32))
        s["frequency"] = _up(np.where(some[2], rng.uniform(0.0, 0.5, rows), 0.0).astype(np.float32))
    if c["bias"]:
        counts = rng.randint(0, min(c["bias"], vocab) + 1, rows)
        counts[0] = min(c["bias"], vocab)
        s["bias_tokens"] = _up(np.concatenate([np.sort(rng.choice(vocab, n, replace=False)) for n in counts]).astype(np.int32))
        s["bias_offsets"] = _up(np.concatenate([[0], np.cumsum(counts)]).astype(np.int32))
        s["bias_values"] = torch.randn(int(counts.sum()), generator=gen, device="cuda") * 4.0
    if c["masked"]:
        words = -(-vocab // 32)
        mask = rng.randint(0, 1 << 32, (rows, words), dtype=np.uint64).astype(np.uint32)
        if rows > 4:
            mask[3] = 0  # a grammar that allows nothing
        use = np.where(rng.rand(rows) < 0.75, np.arange(rows), NONE).astype(np.uint32)
        if rows > 4:
            use[3] = 3
        s["mask"], s["mask_rows"] = _up(mask.view(np.int32)), _up(use.view(np.int32))
    if own:
        kk = _package()
        d = kk.LogitsDesc()
        s["out"], s["tokens"] = torch.empty_like(s["logits"]), torch.empty(rows, dtype=torch.int32, device="cuda")
        d.logits, d.logits_stride, d.out, d.out_stride = s["logits"].data_ptr(), vocab, s["out"].data_ptr(), vocab
        d.rows, d.vocab, d.tokens = rows, vocab, s["tokens"].data_ptr()
        for name in ("history", "history_offsets", "prompt_counts", "repetition", "presence", "frequency",
                     "bias_tokens", "bias_values", "bias_offsets", "mask", "mask_rows"):
            if name in s:
                setattr(d, name, s[name].data_ptr())
        d.history_size = len(s["history"]) if c["penalties"] else 0
        d.bias_size = len(s["bias_tokens"]) if c["bias"] else 0
        if c["masked"]:
            d.mask_stride, d.num_masks = s["mask"].shape[1], rows
        s.update(desc=d, call=kk.kernels()["logits_process"], kk=kk)
    return s


# ---- one pass ---------------------------------------------------------------


def run(state):
    op = state["case"]["op"]
    if own:
        rc = state["call"](ctypes.byref(state["desc"]), torch.cuda.current_stream().cuda_stream)
        if rc != 0:
            raise RuntimeError("%s returned %d" % (op, rc))
        if op == "append":
            return {"query": state["q_out"], "pages": state["storage"][:-1]}
        if op == "attention":
            return state["output"]
        return {"logits": state["out"], "tokens": state["tokens"]}
    if op == "append":
        return _plain_append(state)
    return _plain_attention(state) if op == "attention" else _plain_logits(state)


def _plain_append(s):
    c = s["case"]
    rows, dim, half = c["rows"], c["head_dim"], c["rotary"] // 2
    heads = c["q_heads"] + c["kv_heads"]
    inverse = torch.exp(torch.arange(half, device="cuda", dtype=torch.float64) * (-2.0 / c["rotary"] * math.log(10000.0)))
    angle = s["positions"].double()[:, None] * inverse
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    x = s["qkv"].view(rows, -1, dim)
    a, b = x[:, :heads, :half].float(), x[:, :heads, half:2 * half].float()
    turned = torch.cat([a * cos - b * sin, b * cos + a * sin], -1).half()
    turned = torch.cat([turned, x[:, :heads, 2 * half:]], -1)
    word = s["slots"][:, 1]
    active, extent = (word >> 24) != 0, ((word >> 16) & 255) != 0
    q = turned[:, :c["q_heads"]].reshape(rows, -1)
    s["q_out"] = torch.where(active[:, None], q, s["q_out"])
    cap = torch.where(extent, 64, c["page"])
    at = ((s["slots"][:, 0].long() * s["layers"] + s["layer"]) * 2) * cap + (word & 0xFFFF)
    at = torch.where(extent, at + s["n_micro"], at)
    spare = len(s["storage"]) - 1
    s["storage"].index_copy_(0, torch.where(active, at, spare), turned[:, c["q_heads"]:].reshape(rows, -1))
    s["storage"].index_copy_(0, torch.where(active, at + cap, spare), x[:, heads:].reshape(rows, -1))
    return {"query": s["q_out"], "pages": s["storage"][:-1]}


def _plain_attention(s):
    c = s["case"]
    groups, lanes, hkv = c["groups"], c["lanes"], c["kv_heads"]
    ratio = c["q_heads"] // hkv
    q = s["query"].float().view(groups, lanes, hkv, ratio, 64)
    pk = s["storage"][s["prefix_k"]].float().view(groups, -1, hkv, 64)
    pv = s["storage"][s["prefix_v"]].float().view(groups, -1, hkv, 64)
    tk = s["storage"][s["tail_k"]].float().view(groups, lanes, -1, hkv, 64)
    tv = s["storage"][s["tail_v"]].float().view(groups, lanes, -1, hkv, 64)
    counts = torch.arange(tk.shape[2], device="cuda") < s["tail_n"][:, None]
    counts = counts.view(groups, lanes, 1, 1, -1)
    shared = torch.einsum("gnhrd,gthd->gnhrt", q, pk) * s["scale"]
    tail = torch.einsum("gnhrd,gnthd->gnhrt", q, tk) * s["scale"]
    tail = torch.where(counts, tail, -math.inf)
    top = torch.maximum(shared.amax(-1, keepdim=True), tail.amax(-1, keepdim=True))
    shared, tail = torch.exp(shared - top), torch.exp(tail - top)
    total = shared.sum(-1, keepdim=True) + tail.sum(-1, keepdim=True)
    out = torch.einsum("gnhrt,gthd->gnhrd", shared, pv) + torch.einsum("gnhrt,gnthd->gnhrd", tail, tv)
    return (out / total).half().reshape(groups * lanes, -1)


def _row_of(offsets, size):
    """Row that each entry of a ragged list belongs to."""
    return torch.searchsorted(offsets, torch.arange(size, device="cuda", dtype=offsets.dtype), right=True) - 1


def _plain_logits(s):
    c = s["case"]
    rows, vocab = c["rows"], c["vocab"]
    x = s["logits"]
    if c["penalties"]:
        row = _row_of(s["history_offsets"], len(s["history"]))
        where = row * vocab + s["history"]
        given = torch.arange(len(row), device="cuda") - s["history_offsets"][row] >= s["prompt_counts"][row]
        counts = torch.zeros(rows * vocab, device="cuda")
        seen = counts.index_fill(0, where, 1.0).view(rows, vocab) > 0
        counts = counts.index_add_(0, where, given.float()).view(rows, vocab)
        r = s["repetition"][:, None]
        x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
        x = x - s["frequency"][:, None] * counts
        x = torch.where(counts > 0, x - s["presence"][:, None], x)
    if c["bias"]:
        where = _row_of(s["bias_offsets"], len(s["bias_tokens"])) * vocab + s["bias_tokens"]
        x = x + torch.zeros(rows * vocab, device="cuda").index_copy_(0, where, s["bias_values"]).view(rows, vocab)
    ids = torch.arange(vocab, device="cuda")
    if c["masked"]:
        bits = (s["mask"][:, ids // 32] >> (ids % 32).int()) & 1
        x = torch.where((bits != 0) | (s["mask_rows"] == -1)[:, None], x, -math.inf)
    top = x.amax(-1, keepdim=True)
    token = torch.where(x == top, ids, vocab).amin(-1)
    return {"logits": x, "tokens": torch.where(top[:, 0] > -math.inf, token, -1).int()}


# ---- what a pass cannot do without ------------------------------------------


def work(case):
    c = case
    if c["op"] == "append":
        live = c["rows"] - c["padded"]
        q, kv = c["q_heads"] * c["head_dim"], c["kv_heads"] * c["head_dim"]
        return {"bytes": live * (4 * q + 8 * kv + 4) + 8 * c["rows"],
                "flops": live * 3 * c["rotary"] * (c["q_heads"] + c["kv_heads"])}
    if c["op"] == "attention":
        n = c["groups"] * c["lanes"]
        tails = c["lanes"] * (c["lanes"] + 1) // 2 * c["groups"] if c["chunk"] else n * c["suffix"] / 2
        read = c["groups"] * c["lanes"] if c["chunk"] else tails
        return {"bytes": (c["groups"] * c["prefix"] + read) * c["kv_heads"] * 256 + n * c["q_heads"] * 256,
                "flops": 256 * c["q_heads"] * (n * c["prefix"] + tails)}
    size = c["rows"] * c["vocab"]
    history = c["rows"] * c["history"] * 5 / 8 if c["penalties"] else 0
    return {"bytes": 8 * size + 4 * history + 4 * c["rows"] * c["bias"] + (size / 8 if c["masked"] else 0),
            "flops": size + 4 * history}


# ---- the definitions in 64 bits ---------------------------------------------


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attention": _exact_attention, "logits": _exact_logits}[case["op"]](s, case)


def _page_views(s, c, storage):
    n = s["n_micro"]
    shape = (s["layers"], 2, -1, c["kv_heads"], s["head_dim"])
    micro = storage[:n].view(s["micro"], *shape[:2], c["page"], *shape[3:])
    extent = storage[n:-1].view(s["extent"], *shape[:2], 64, *shape[3:])
    return micro, extent


def _exact_append(s, c):
    dim, hq, hkv, rot = c["head_dim"], c["q_heads"], c["kv_heads"], c["rotary"]
    x = s["qkv"].double().view(c["rows"], hq + 2 * hkv, dim)
    power = torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot
    turn = torch.polar(torch.ones(c["rows"], rot // 2, device="cuda", dtype=torch.float64),
                       s["positions"].double()[:, None] / 10000.0 ** power)
    storage = s["storage"].double()
    micro, extent = _page_views(s, c, storage)
    q_out = s["q_out"].double()
    on = torch.from_numpy(s["host_slots"][:, 1] >> 24 != 0).cuda()
    z = torch.complex(x[:, :hq + hkv, :rot // 2], x[:, :hq + hkv, rot // 2:rot]) * turn[:, None]
    x[:, :hq + hkv, :rot // 2], x[:, :hq + hkv, rot // 2:rot] = z.real, z.imag
    q_out[on] = x[on, :hq].reshape(int(on.sum()), -1)
    for pool, kind in ((micro, 0), (extent, 1)):
        pick = np.nonzero((s["host_slots"][:, 1] >> 24 != 0) & ((s["host_slots"][:, 1] >> 16 & 255) == kind))[0]
        slot, token = s["host_slots"][pick, 0].astype(np.int64), s["host_slots"][pick, 1].astype(np.int64) & 0xFFFF
        rows, slot, token = _up(pick), _up(slot), _up(token)
        pool[slot, s["layer"], 0, token] = x[rows, hq:hq + hkv]
        pool[slot, s["layer"], 1, token] = x[rows, hq + hkv:]
    return {"query": q_out, "pages": storage[:-1]}


def _exact_attention(s, c):
    micro, extent = _page_views(s, c, s["storage"])
    ratio = c["q_heads"] // c["kv_heads"]
    out = torch.empty(s["query"].shape, dtype=torch.float64, device="cuda")

    def read(table):
        parts = [(extent if kind else micro)[slot, s["layer"], :, :n] for slot, _, n, kind in table.tolist()]
        return torch.cat(parts, 1).double() if parts else torch.zeros(2, 0, c["kv_heads"], 64, device="cuda", dtype=torch.float64)

    heads = [None, None]
    shared = int((np.cumsum(s["tables"][0][:, 2]) <= c["prefix"]).sum())
    for b, table in enumerate(s["tables"]):
        if heads[0] != b // c["lanes"]:
            heads = [b // c["lanes"], read(table[:shared])]
        kv = torch.cat([heads[1], read(table[shared:])], 1)
        q = s["query"][b].double().view(c["kv_heads"], ratio, 64)
        score = torch.matmul(q, kv[0].permute(1, 2, 0)) / 8.0
        weight = torch.softmax(score, -1)
        out[b] = torch.matmul(weight, kv[1].permute(1, 0, 2)).reshape(-1)
    return out


def _exact_logits(s, c):
    out = s["logits"].double()
    host = {k: v.cpu().numpy() for k, v in s.items() if isinstance(v, torch.Tensor) and k != "logits"}
    for r in range(c["rows"]):
        row = out[r]
        if c["penalties"]:
            text = host["history"][host["history_offsets"][r]:host["history_offsets"][r + 1]]
            seen = torch.from_numpy(np.unique(text).astype(np.int64)).cuda()
            v = row[seen]
            p = float(host["repetition"][r])
            row[seen] = torch.where(v > 0, v / p, v * p)
            ids, n = np.unique(text[host["prompt_counts"][r]:], return_counts=True)
            ids = torch.from_numpy(ids.astype(np.int64)).cuda()
            row[ids] -= float(host["frequency"][r]) * torch.from_numpy(n).cuda().double() + float(host["presence"][r])
        if c["bias"]:
            lo, hi = host["bias_offsets"][r:r + 2]
            ids = torch.from_numpy(host["bias_tokens"][lo:hi].astype(np.int64)).cuda()
            row[ids] += torch.from_numpy(host["bias_values"][lo:hi]).cuda().double()
        if c["masked"] and host["mask_rows"][r] != -1:
            bits = np.unpackbits(host["mask"][host["mask_rows"][r]].view(np.uint8), bitorder="little")[:c["vocab"]]
            row[torch.from_numpy(bits == 0).cuda()] = -math.inf
    return {"logits": out, "tokens": None}
