"""A serving step as its operators make it, one after the other on one stream: a
ragged prompt batch is rotated and written into pages, lanes fork from the two
prompts, and every decode step appends a token per lane, groups and plans the
lanes, attends, projects onto the vocabulary and picks the lanes' next tokens.
Each stage is held against a 64-bit reference of what the stage before left on
the device."""
import ctypes as C
import random

import numpy as np
import pytest
import torch

from gpu_util import p, to_device_bytes
from test_kv_append import assert_rounded, rotate_ref
from test_logits import Case
from test_prefix_attention import find, pack, plan_for

pytestmark = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]

DIM, THETA = 64, 10000.0


class Server:
    """Pages, lanes and weights; `tables` holds a lane's (slot, begin, valid, kind) entries."""

    def __init__(self, kk, hq, hkv, page, vocab, seed):
        self.kk, self.K, self.hq, self.hkv, self.page, self.vocab = kk, kk.kernels(), hq, hkv, page, vocab
        self.rng, self.np = random.Random(seed), np.random.RandomState(seed)
        self.layers, self.layer, self.next = 2, 1, [0, 0]
        nan = float("nan")
        self.micro = torch.full((160, self.layers, 2, page, hkv, DIM), nan, dtype=torch.half, device="cuda")
        self.extent = torch.full((40, self.layers, 2, 64, hkv, DIM), nan, dtype=torch.half, device="cuda")
        self.pools = kk.KvPools(p(self.micro), p(self.extent), 160, 40, self.layers, hkv, DIM, page)
        width = (hq + 2 * hkv) * DIM
        self.qkv = (self.np.randn(vocab, width) * 1.2).astype(np.float16)  # what a token projects to
        self.head = torch.from_numpy((self.np.randn(vocab, hq * DIM) * 0.5).astype(np.float16)).cuda()
        self.keys = {}  # (kind, slot, token) -> rows that were written there
        self.values = {}

    def extend(self, table, tokens, extents):
        """Room for `tokens` more of a lane: their slots, and the table with them."""
        table, slots = list(table), []
        at = sum(e[2] for e in table)
        for i in range(tokens):
            last = table[-1] if table else None
            if last is None or last[2] == (64 if last[3] else self.page):
                kind = int(extents and tokens - i >= 64)
                table.append((self.next[kind], at + i, 0, kind))
                self.next[kind] += 1
                last = table[-1]
            slots.append((last[0], last[2], last[3]))
            table[-1] = (last[0], last[1], last[2] + 1, last[3])
        return table, slots

    def append(self, ids, positions, slots, active):
        rows, hq, hkv = len(ids), self.hq, self.hkv
        x = self.qkv[np.asarray(ids)]
        x[~np.asarray(active)] = np.nan
        self.x = torch.from_numpy(x).cuda()
        self.q = torch.full((rows, hq * DIM), float("nan"), dtype=torch.half, device="cuda")
        d = self.kk.KvAppendDesc()
        d.pools, d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = self.pools, self.layer, rows, hq, DIM, THETA
        self.d_slots = to_device_bytes((self.kk.KvSlot * rows)(
            *[self.kk.KvSlot(s, t, k, int(a)) for (s, t, k), a in zip(slots, active)]))
        self.d_positions = torch.tensor(positions, dtype=torch.int32, device="cuda")
        d.slots, d.positions = p(self.d_slots), p(self.d_positions)
        d.query, d.key, d.value = (p(self.x) + 2 * DIM * n for n in (0, hq, hq + hkv))
        d.query_stride = d.key_stride = d.value_stride = x.shape[1]
        d.query_out, d.query_out_stride = p(self.q), hq * DIM
        return d

    def check_append(self, ids, positions, slots, active):
        torch.cuda.synchronize()
        live = np.flatnonzero(active)
        x = self.qkv[np.asarray(ids)[live]].reshape(len(live), -1, DIM)
        pools = (self.micro[:, self.layer].cpu().numpy(), self.extent[:, self.layer].cpu().numpy())
        k = np.stack([pools[slots[i][2]][slots[i][0], 0, slots[i][1]] for i in live])
        v = np.stack([pools[slots[i][2]][slots[i][0], 1, slots[i][1]] for i in live])
        got = np.concatenate([self.q.cpu().numpy()[live].reshape(len(live), self.hq, DIM), k], 1)
        turned = x[:, :self.hq + self.hkv]
        half = np.abs(turned[..., :DIM // 2].astype(float)) + np.abs(turned[..., DIM // 2:].astype(float))
        assert_rounded(got, rotate_ref(turned, np.asarray(positions)[live], DIM, THETA), np.concatenate([half, half], -1))
        assert np.array_equal(v, x[:, self.hq + self.hkv:])
        assert bool(torch.isnan(self.q[torch.from_numpy(~np.asarray(active)).cuda()]).all())
        for pool in (self.micro, self.extent):  # the other layer
            assert bool(torch.isnan(pool[:, 1 - self.layer]).all())

    def attention(self, tables):
        kk, B = self.kk, len(tables)
        descs, lanes, nd = pack(kk, tables)
        groups, ng = find(kk, descs, lanes, B)
        rc, items, plan = plan_for(kk, descs, nd, lanes, B, groups, ng, self.hq, self.hkv, 148)
        assert rc == 0
        self.groups_found = ng
        self.tables_on_device = [to_device_bytes(a) for a in (
            descs, lanes, groups, (kk.PrefixItem * max(1, plan.num_items))(*items[:plan.num_items]))]
        size = self.K["prefix_attention_workspace_bytes"](C.byref(plan))
        self.workspace = torch.empty(max(16, size), dtype=torch.uint8, device="cuda")
        self.out = torch.empty(B, self.hq * DIM, dtype=torch.half, device="cuda")
        d = kk.PrefixAttnDesc()
        d.pools, d.layer, d.q_heads, d.scale, d.plan = self.pools, self.layer, self.hq, DIM ** -0.5, plan
        d.descs, d.lanes, d.groups, d.items = map(p, self.tables_on_device)
        d.query, d.query_stride, d.output, d.output_stride = p(self.q), self.hq * DIM, p(self.out), self.hq * DIM
        d.workspace, d.workspace_bytes = p(self.workspace), size
        return d

    def check_attention(self, tables):
        for b, t in enumerate(tables):
            k, v = torch.cat([(self.extent if kind else self.micro)[s, self.layer, :, :n] for s, _, n, kind in t], 1).double()
            q = self.q[b].double().view(self.hkv, -1, DIM)
            score = torch.einsum("hgd,thd->hgt", q, k) * DIM ** -0.5
            ref = torch.einsum("hgt,thd->hgd", torch.softmax(score, -1), v).reshape(-1)
            top = float(torch.einsum("hgd,thd->hgt", q.abs(), k.abs()).max()) * DIM ** -0.5
            # FP32 scores of 64 products: a weight is off by 2^-17 top; 2^-21 for its exponential;
            # twice that in a quotient. A shared token's weight in FP16: 2^-11. A sum over T tokens:
            # 2^-23 a token. All of the largest value; and half an FP16 step of the result.
            size = float(v.abs().max()) * (2 * (top * 2.0 ** -17 + 2.0 ** -21) + 2.0 ** -11 + (k.shape[0] + 64) * 2.0 ** -23)
            over = (self.out[b].double() - ref).abs() - (ref.abs() * 2.0 ** -11 + 2.0 ** -25 + size)
            assert float(over.max()) <= 0, f"lane {b}"

    def project(self, rows):
        self.logits = torch.full((rows, self.vocab), float("nan"), device="cuda")
        d = self.kk.GemmDesc()
        d.weight, d.M, d.K = p(self.head), self.vocab, self.hq * DIM
        d.x, d.N, d.x_stride, d.x_rows = p(self.out), rows, self.hq * DIM, rows
        d.epilogue, d.out, d.out_stride = self.kk.EPI_STORE_F32, p(self.logits), self.vocab
        return d

    def check_project(self):
        x, w = self.out.double(), self.head.double()
        bound = (x.abs() @ w.abs().T) * (x.shape[1] * 2.0 ** -23)  # FP32 sums of K products, a rounding each
        assert bool(((self.logits.double() - x @ w.T).abs() <= bound).all())

    def choose(self, texts, prompts):
        rows = len(texts)
        c = self.case = Case(rows, self.vocab, seed=len(texts[0]))
        c.history, c.prompts = [np.asarray(t, np.uint32) for t in texts], np.asarray(prompts, np.uint32)
        c.factors = [np.full(rows, f, np.float32) for f in (1.3, 0.4, 0.2)]
        c.with_bias([5] * rows)
        c.with_mask(0.7, 2, [0, 1, 0xFFFFFFFF] * rows)
        c.mask_rows = c.mask_rows[:rows]
        flat = lambda lists, dtype: torch.from_numpy(np.concatenate(lists).astype(dtype)).cuda()  # noqa: E731
        ends = lambda lists: torch.tensor(np.cumsum([0] + [len(t) for t in lists]), dtype=torch.int32).cuda()  # noqa: E731
        ids, values = [b[0] for b in c.bias], [b[1] for b in c.bias]
        self.kept = keep = [flat(c.history, np.int32), ends(c.history), torch.tensor(prompts, dtype=torch.int32).cuda(),
                            *[torch.from_numpy(f).cuda() for f in c.factors], flat(ids, np.int32), flat(values, np.float32),
                            ends(ids), torch.from_numpy(c.mask.view(np.int32)).cuda(),
                            torch.from_numpy(c.mask_rows.view(np.int32)).cuda()]
        self.tokens = torch.empty(rows, dtype=torch.int32, device="cuda")
        self.processed = torch.empty_like(self.logits)
        d = self.kk.LogitsDesc()
        d.logits, d.logits_stride, d.rows, d.vocab = p(self.logits), self.vocab, rows, self.vocab
        d.out, d.out_stride, d.tokens = p(self.processed), self.vocab, p(self.tokens)
        (d.history, d.history_offsets, d.prompt_counts, d.repetition, d.presence, d.frequency,
         d.bias_tokens, d.bias_values, d.bias_offsets, d.mask, d.mask_rows) = map(p, keep)
        d.history_size, d.bias_size = len(keep[0]), len(keep[6])
        d.mask_stride, d.num_masks = c.mask.shape[1], 2
        return d

    def check_choose(self):
        self.case.logits = self.logits.cpu().numpy()
        x, want = self.case.expect()
        assert np.array_equal(self.processed.cpu().numpy(), x)
        tokens = self.tokens.cpu().numpy()
        assert np.array_equal(tokens, want)
        return [int(t) for t in tokens]


@pytest.mark.parametrize("hq,hkv,page,extents", [(32, 4, 8, True), (6, 2, 16, False), (8, 8, 8, True)], ids=str)
def test_decode_steps_of_forked_lanes(kk, hq, hkv, page, extents):
    s = Server(kk, hq, hkv, page, 1003, hq)
    rng = s.rng
    prompts = [[rng.randrange(s.vocab) for _ in range(n)] for n in (333, 70)]
    # Prompts: one ragged batch, with rows behind the last sequence that are padding.
    tables, slots = zip(*[s.extend([], len(t), extents) for t in prompts])
    ids = prompts[0] + prompts[1] + [0] * 13
    positions = [i for t in prompts for i in range(len(t))] + [0] * 13
    places = slots[0] + slots[1] + [(0, 0, 0)] * 13
    active = [True] * (len(ids) - 13) + [False] * 13
    d = s.append(ids, positions, places, active)
    assert s.K["kv_append_rope"](C.byref(d), None) == 0
    s.check_append(ids, positions, places, active)

    # Forks: a lane's own tokens go into pages of its own (the prompt's last page stays as it is).
    owner = [0, 0, 0, 1, 1, 0, 0]
    shared = [list(tables[o]) for o in owner]
    own = [[] for _ in owner]
    texts = [list(prompts[o]) for o in owner]
    last = [rng.randrange(s.vocab) for _ in owner]
    stream = torch.cuda.Stream()
    for step in range(10):
        rows = len(owner)
        places, positions = [], []
        for b in range(rows):
            texts[b].append(last[b])
            begin = len(prompts[owner[b]])
            own[b], place = s.extend(own[b], 1, False)
            places += place
            positions.append(begin + sum(e[2] for e in own[b]) - 1)
        full = [sh + [(sl, len(prompts[o]) + at, n, k) for sl, at, n, k in ow] for sh, ow, o in zip(shared, own, owner)]
        calls = [("kv_append_rope", s.append(last, positions, places, [True] * rows)),
                 ("prefix_attention", s.attention(full)), ("gemm", s.project(rows)),
                 ("logits_process", s.choose(texts, [len(prompts[o]) for o in owner]))]
        assert s.groups_found == 3

        def run(on):
            for name, desc in calls:
                assert s.K[name](C.byref(desc), on) == 0, name

        torch.cuda.synchronize()
        s.K["set_pdl"](step % 2)
        run(stream.cuda_stream)
        s.K["set_pdl"](0)
        torch.cuda.synchronize()
        assert s.K["device_status"](None) == 0
        s.check_append(last, positions, places, [True] * rows)
        s.check_attention(full)
        s.check_project()
        chosen = s.check_choose()
        if step % 4 == 0:  # the step as one graph, twice: the same bits
            kept = [t.clone() for t in (s.q, s.out, s.logits, s.processed, s.tokens)]
            # Launched ahead of each other's ends as well (programmatic dependents).
            s.K["set_pdl"](int(step > 0))
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=stream):
                run(stream.cuda_stream)
            s.K["set_pdl"](0)
            for _ in range(2):
                for t in (s.q, s.out, s.logits, s.processed, s.tokens):
                    t.fill_(3)
                graph.replay()
                torch.cuda.synchronize()
                assert s.K["device_status"](None) == 0
                for t, k in zip((s.q, s.out, s.logits, s.processed, s.tokens), kept):
                    assert torch.equal(t, k)
        last = [t if t >= 0 else 0 for t in chosen]
