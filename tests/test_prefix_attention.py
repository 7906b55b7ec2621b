"""kk_prefix_attention: decode attention of lanes that share a prefix. Grouping,
planning and refusals run on the CPU; the numerics run on the GPU against a
64-bit reference over the same pages."""
import ctypes as C
import random

import pytest
import torch

from gpu_util import p, to_device_bytes

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]


def gpu_test(fn):
    for mark in gpu:
        fn = mark(fn)
    return fn


# ---- tables -----------------------------------------------------------------


class Pages:
    def __init__(self, rng, page=8):
        self.rng, self.page, self.next = rng, page, [0, 0]

    def take(self, kind):
        self.next[kind] += 1
        return self.next[kind] - 1

    def table(self, tokens, begin=0, ragged=False, extents=True):
        """(slot, begin, valid, kind) entries; `ragged`: pages are left partly filled."""
        out, t = [], 0
        while t < tokens:
            kind = 1 if extents and self.page == 8 and tokens - t >= 64 and self.rng.random() < 0.8 else 0
            cap = 64 if kind else self.page
            n = min(cap, tokens - t)
            if ragged and self.rng.random() < 0.3:
                n = self.rng.randint(1, n)
            out.append((self.take(kind), begin + t, n, kind))
            t += n
        return out


def pack(kk, tables):
    flat = [e for t in tables for e in t]
    descs = (kk.PageDesc * max(1, len(flat)))(*[kk.PageDesc(s, b, n, k, 0, 0) for s, b, n, k in flat])
    lanes = (kk.AttnLane * max(1, len(tables)))()
    at = 0
    for b, t in enumerate(tables):
        lanes[b].desc_offset, lanes[b].desc_count = at, len(t)
        lanes[b].token_count, lanes[b].query_row = sum(e[2] for e in t), b
        at += len(t)
    return descs, lanes, len(flat)


def find(kk, descs, lanes, n, min_lanes=2, min_tokens=1):
    groups = (kk.PrefixGroup * max(1, n))()
    count = kk.kernels()["prefix_groups"](descs, lanes, n, min_lanes, min_tokens, groups, n)
    return groups, count


def plan_for(kk, descs, nd, lanes, nl, groups, ng, hq, hkv, sms=148, room=65536):
    items, plan = (kk.PrefixItem * room)(), kk.PrefixPlan()
    rc = kk.kernels()["prefix_attention_plan"](descs, nd, lanes, nl, groups, ng, hq, hkv, sms, items, room, C.byref(plan))
    return rc, items, plan


# ---- grouping and planning (CPU) ---------------------------------------------


def test_groups_of_forks(kk):
    pages = Pages(random.Random(1))
    a, b = pages.table(200), pages.table(70)
    tails = [pages.table(n, 200) for n in (0, 5, 64, 1)]
    tables = [a + t for t in tails] + [b + pages.table(9, 70), b, pages.table(300), [], a + pages.table(3, 200)]
    descs, lanes, nd = pack(kk, tables)
    groups, n = find(kk, descs, lanes, len(tables), min_tokens=64)
    assert n == 2
    assert (groups[0].lane_begin, groups[0].lane_count, groups[0].token_count, groups[0].desc_count) == (0, 4, 200, len(a))
    assert (groups[1].lane_begin, groups[1].lane_count, groups[1].token_count, groups[1].desc_count) == (4, 2, 70, len(b))
    assert [lanes[i].token_count for i in range(9)] == [0, 5, 64, 1, 9, 0, 300, 0, 203]
    assert [lanes[i].desc_count for i in range(4)] == [len(t) for t in tails]
    # Too few lanes or tokens: nothing is cut off.
    for kw in (dict(min_lanes=5), dict(min_tokens=201)):
        descs, lanes, nd = pack(kk, tables)
        assert find(kk, descs, lanes, len(tables), **kw)[1] == 0
        assert lanes[0].token_count == 200 and lanes[0].desc_offset == 0


def test_groups_differ_by_valid_tokens_and_stop_at_room(kk):
    tables = [[(0, 0, 64, 1), (0, 64, 3, 0)], [(0, 0, 64, 1), (0, 64, 4, 0)], [(1, 0, 8, 0)], [(1, 0, 8, 0)]]
    descs, lanes, nd = pack(kk, tables)
    groups, n = find(kk, descs, lanes, 4)
    assert n == 2 and groups[0].token_count == 64 and lanes[0].token_count == 3
    descs, lanes, nd = pack(kk, tables)
    groups = (kk.PrefixGroup * 1)()
    assert kk.kernels()["prefix_groups"](descs, lanes, 4, 2, 1, groups, 1) == 1
    assert lanes[2].token_count == 8
    for empty in (0, 1):
        assert kk.kernels()["prefix_groups"](descs, lanes, empty, 2, 1, groups, 1) == 0


def own_tokens(lanes, n):
    return sum(lanes[i].token_count for i in range(n))


@pytest.mark.parametrize("at", [0, 5, 31, 63])
def test_groups_with_a_short_lane_among_long_ones(kk, at):
    """A lane that holds only the first page of what the others share does not cut their sharing down to it."""
    pages = Pages(random.Random(30))
    shared = pages.table(64) + pages.table(4096, 64)
    tables = [shared[:1] if i == at else shared + pages.table(i, 4160) for i in range(64)]
    assert shared[0][2] == 64
    descs, lanes, nd = pack(kk, tables)
    groups, n = find(kk, descs, lanes, 64, min_tokens=64)
    assert n == (2 if at in (5, 31) else 1)
    for g in range(n):
        assert groups[g].token_count == 4160 and groups[g].desc_count == len(shared)
    assert sum(groups[g].lane_count for g in range(n)) == 63
    assert own_tokens(lanes, 64) == sum(i for i in range(64) if i != at) + 64


def test_groups_of_pairs_that_share_a_little_more(kk):
    """Lanes that share a long prompt, every two of them some tokens behind it: the prompt is read once."""
    pages = Pages(random.Random(31))
    prompt = pages.table(2000)
    tables = []
    for _ in range(16):
        more = prompt + pages.table(100, 2000)
        tables += [more + pages.table(3, 2100), more + pages.table(9, 2100)]
    descs, lanes, nd = pack(kk, tables)
    groups, n = find(kk, descs, lanes, 32)
    assert n == 1 and (groups[0].lane_begin, groups[0].lane_count, groups[0].token_count) == (0, 32, 2000)
    # Pairs that share much more than the prompt stand alone.
    tables = []
    for _ in range(4):
        more = prompt[:4] + pages.table(9000, 256)
        tables += [more + pages.table(3, 9256), more + pages.table(9, 9256)]
    descs, lanes, nd = pack(kk, tables)
    assert find(kk, descs, lanes, 8)[1] == 4


@pytest.mark.parametrize("seed", range(40))
def test_groups_have_the_largest_gain(kk, seed):
    """Against every way to cut the lanes into runs. A run of n lanes gains (n - 1) x (shared tokens + 1375)."""
    rng = random.Random(seed)
    pages = Pages(rng)
    n = rng.randint(1, 9)
    pieces = [[pages.table(rng.choice([1, 8, 64, 200, 3000])) for _ in range(2)] for _ in range(4)]
    tables = []
    for _ in range(n):
        t = []
        for p_ in pieces[:rng.randint(0, 4)]:
            t += p_[int(rng.random() < 0.2)]
        tables.append(t + (pages.table(rng.randint(1, 70)) if rng.random() < 0.7 else []))
    if rng.random() < 0.5:
        tables.sort(key=lambda t: [e[:1] + e[2:] for e in t])
    min_lanes, min_tokens = rng.choice([0, 2, 2, 3, 4]), rng.choice([0, 1, 64, 250])

    def shared(b, e):
        count = 0
        while all(count < len(t) for t in tables[b:e]) and len({t[count][:1] + t[count][2:] for t in tables[b:e]}) == 1:
            count += 1
        return count, sum(x[2] for x in tables[b][:count])

    def gain(b, e):
        tokens = shared(b, e)[1]
        return (e - b - 1) * (tokens + 1375) if e - b >= max(2, min_lanes) and tokens >= max(1, min_tokens) else 0

    best = [0] * (n + 1)
    for e in range(1, n + 1):
        best[e] = max(best[b] + gain(b, e) for b in range(e))
    descs, lanes, nd = pack(kk, tables)
    before = [(lanes[b].desc_offset, lanes[b].desc_count, lanes[b].token_count) for b in range(n)]
    groups, ng = find(kk, descs, lanes, n, min_lanes, min_tokens)
    end, total = 0, 0
    grouped = {}
    for g in groups[:ng]:
        assert g.lane_begin >= end and gain(g.lane_begin, g.lane_begin + g.lane_count) > 0
        end = g.lane_begin + g.lane_count
        assert (g.desc_count, g.token_count) == shared(g.lane_begin, end) and g.desc_offset == before[g.lane_begin][0]
        total += gain(g.lane_begin, end)
        grouped.update({b: g for b in range(g.lane_begin, end)})
    assert end <= n and total == best[n]
    for b in range(n):
        cut = (grouped[b].desc_count, grouped[b].token_count) if b in grouped else (0, 0)
        assert (lanes[b].desc_offset, lanes[b].desc_count, lanes[b].token_count) == (
            before[b][0] + cut[0], before[b][1] - cut[0], before[b][2] - cut[1])


def tile_fill(entries):
    """128-token tiles of a run as the kernel fills them: 16 groups of 8 tokens, pages whole."""
    tiles, n = 0, 0
    for _, _, valid, _ in entries:
        g = -(-valid // 8)
        if n + g > 16:
            tiles, n = tiles + 1, 0
        n += g
    return tiles + (n > 0)


@pytest.mark.parametrize("seed", range(8))
@pytest.mark.parametrize("sms", [1, 7, 148])
def test_plan_covers_every_page_once(kk, seed, sms):
    rng = random.Random(seed)
    pages = Pages(rng, rng.choice([8, 8, 16, 64]))
    hkv = rng.choice([1, 3, 4, 8])
    hq = hkv * rng.choice([1, 3, 8, 16])
    tables = []
    for _ in range(rng.randint(1, 4)):
        shared = pages.table(rng.choice([1, 64, 130, 1000, 6000]), ragged=rng.random() < 0.5)
        tables += [shared + pages.table(rng.choice([0, 1, 9, 64, 700]), ragged=rng.random() < 0.5)
                   for _ in range(rng.choice([1, 2, 5, 40]))]
    descs, lanes, nd = pack(kk, tables)
    groups, ng = find(kk, descs, lanes, len(tables))
    rc, items, plan = plan_for(kk, descs, nd, lanes, len(tables), groups, ng, hq, hkv, sms)
    assert rc == 0 and plan.num_lanes == len(tables) and plan.num_groups == ng and plan.num_descs == nd
    flat = [e for t in tables for e in t]
    G = hq // hkv
    used = []   # partial rows, as intervals
    shared = {}
    for i in range(plan.num_shared):
        it = items[i]
        assert it.row_tiles in (1, 2) and it.token_tiles == tile_fill(flat[it.desc_begin:it.desc_end])
        shared.setdefault((it.owner, it.kv_head, it.row_tile, it.row_tiles), []).append(it)
    for g in range(ng):
        grp = groups[g]
        rows = grp.lane_count * G
        assert grp.row_tiles == -(-rows // 128)
        for h in range(hkv):
            at = 0
            while at < grp.row_tiles:
                tiles = min(2, grp.row_tiles - at)
                run = shared.pop((g, h, at, tiles))
                assert [r.part for r in run] == list(range(grp.part_count))
                assert [r.part_row for r in run] == [grp.part_row + ((h * grp.part_count + i) * grp.row_tiles + at) * 128
                                                     for i in range(grp.part_count)]
                assert all((r.lane_begin, r.lane_count) == (grp.lane_begin, grp.lane_count) for r in run)
                edges = [r.desc_begin for r in run] + [run[-1].desc_end]
                assert edges[0] == grp.desc_offset and edges[-1] == grp.desc_offset + grp.desc_count
                assert all(r.desc_end == e for r, e in zip(run, edges[1:]))
                at += tiles
        used.append((grp.part_row, grp.part_row + hkv * grp.part_count * grp.row_tiles * 128))
        assert all(lanes[b].reserved == g + 1 for b in range(grp.lane_begin, grp.lane_begin + grp.lane_count))
    assert not shared
    own = {}
    for i in range(plan.num_shared, plan.num_items):
        it = items[i]
        assert it.row_tiles == 0
        own.setdefault((it.owner, it.kv_head), []).append(it)
    for b in range(len(tables)):
        ln = lanes[b]
        tokens = sum(flat[e][2] for e in range(ln.desc_offset, ln.desc_offset + ln.desc_count))
        assert (ln.item_count > 0) == (tokens > 0)
        for h in range(hkv):
            run = own.pop((b, h), [])
            assert [r.part for r in run] == list(range(ln.item_count))
            assert [r.part_row for r in run] == [ln.item_offset + i * hq + h * G for i in range(ln.item_count)]
            if run:
                edges = [r.desc_begin for r in run] + [run[-1].desc_end]
                assert edges[0] == ln.desc_offset and edges[-1] == ln.desc_offset + ln.desc_count
                assert all(r.desc_end == e for r, e in zip(run, edges[1:]))
        used.append((ln.item_offset, ln.item_offset + ln.item_count * hq))
    assert not own
    used = sorted(u for u in used if u[0] != u[1])
    assert all(a[1] == b[0] for a, b in zip(used, used[1:]))  # no row twice, none left out
    assert (used[-1][1] if used else 0) == plan.part_rows
    assert kk.kernels()["prefix_attention_workspace_bytes"](C.byref(plan)) == plan.part_rows * 264
    # Items beyond the room are counted, not written.
    if plan.num_items > 3:
        few, small = (kk.PrefixItem * 4)(), kk.PrefixPlan()
        few[3].owner = 77
        rc = kk.kernels()["prefix_attention_plan"](descs, nd, lanes, len(tables), groups, ng, hq, hkv, sms, few, 3, C.byref(small))
        assert rc == 0 and small.num_items == plan.num_items and few[3].owner == 77


def test_plan_refuses_descriptors_behind_the_end(kk):
    """Every lane and the group reach to some last descriptor: one fewer is refused, as many are enough."""
    pages = Pages(random.Random(34))
    shared = pages.table(100)
    for tails in ([0, 0, 0], [5, 0, 9], [0, 70, 0], [3, 3, 3]):
        tables = [shared + pages.table(n, 100) for n in tails]
        for grouped in (True, False):
            descs, lanes, nd = pack(kk, tables)
            groups, ng = find(kk, descs, lanes, 3) if grouped else ((kk.PrefixGroup * 1)(), 0)
            assert ng == int(grouped)
            assert plan_for(kk, descs, nd, lanes, 3, groups, ng, 32, 4)[0] == 0
            assert plan_for(kk, descs, nd - 1, lanes, 3, groups, ng, 32, 4)[0] == kk.KK_EINVAL
            if not grouped:
                continue
            # The lanes' own tables inside, the group's run one too long.
            groups[0].desc_offset, groups[0].desc_count = nd - 2, 3
            assert plan_for(kk, descs, nd, lanes, 3, groups, 1, 32, 4)[0] == kk.KK_EINVAL
            groups[0].desc_count = 2
            assert plan_for(kk, descs, nd, lanes, 3, groups, 1, 32, 4)[0] == 0


@pytest.mark.parametrize("groups,lanes,prefix,own,hkv", [
    (16, 4, 300, 1000, 8), (18, 2, 64, 1000, 8), (19, 2, 64, 1000, 8), (32, 4, 300, 1000, 8), (36, 2, 300, 500, 4),
    (40, 2, 300, 500, 4), (128, 2, 64, 64, 8), (1, 4096, 256, 30, 4), (9, 3, 3000, 700, 8),
])
def test_plan_spreads_own_pages_beside_many_prefixes(kk, groups, lanes, prefix, own, hkv):
    """As many prefixes, times KV heads and row tiles, as there are SMs and more: what the lanes have of their own
    is spread over many thread blocks all the same."""
    rng = random.Random(groups)
    pages = Pages(rng)
    tables = []
    for _ in range(groups):
        tables += forks(pages, prefix, [rng.randint(0, own) for _ in range(lanes)])
    descs, lane_array, nd = pack(kk, tables)
    group_array, ng = find(kk, descs, lane_array, len(tables))
    assert ng == groups
    rc, items, plan = plan_for(kk, descs, nd, lane_array, len(tables), group_array, ng, 4 * hkv, hkv)
    assert rc == 0 and plan.num_items <= 65536
    flat = [e for t in tables for e in t]
    work = [sum(flat[e][2] for e in range(it.desc_begin, it.desc_end)) for it in items[plan.num_shared:plan.num_items]]
    blocks = [sum(work[i:i + plan.tasks_per_cta]) for i in range(0, len(work), plan.tasks_per_cta)]
    assert max(blocks) <= 4 * sum(work) / 148 + 8 * 64


def test_plan_refuses(kk):
    pages = Pages(random.Random(3))
    shared = pages.table(100)

    def fresh():
        descs, lanes, nd = pack(kk, [shared + pages.table(5, 100), list(shared), list(shared)])
        groups, ng = find(kk, descs, lanes, 3)
        assert ng == 1
        return descs, nd, lanes, groups

    descs, nd, lanes, groups = fresh()
    assert plan_for(kk, descs, nd, lanes, 3, groups, 1, 32, 4)[0] == 0
    for hq, hkv, sms in ((30, 4, 148), (32, 0, 148), (0, 4, 148), (17, 1, 148), (32, 4, 0), (8192, 512, 148)):
        assert plan_for(kk, descs, nd, lanes, 3, groups, 1, hq, hkv, sms)[0] == kk.KK_EINVAL
    assert plan_for(kk, descs, nd - 1, lanes, 3, groups, 1, 32, 4)[0] == 0 or lanes[2].desc_count == 0
    for change in (dict(lane_count=3 + 1), dict(lane_begin=4), dict(desc_count=nd + 1), dict(desc_offset=nd + 1),
                   dict(desc_offset=0xFFFFFFFF, desc_count=2), dict(lane_begin=0xFFFFFFFF, lane_count=2)):
        descs, nd, lanes, groups = fresh()
        for k_, v in change.items():
            setattr(groups[0], k_, v)
        assert plan_for(kk, descs, nd, lanes, 3, groups, 1, 32, 4)[0] == kk.KK_EINVAL
    descs, nd, lanes, groups = fresh()
    two = (kk.PrefixGroup * 2)(groups[0], groups[0])  # every lane twice
    assert plan_for(kk, descs, nd, lanes, 3, two, 2, 32, 4)[0] == kk.KK_EINVAL
    descs, nd, lanes, groups = fresh()
    lanes[1].desc_offset, lanes[1].desc_count = nd, 1
    assert plan_for(kk, descs, nd, lanes, 3, groups, 1, 32, 4)[0] == kk.KK_EINVAL
    assert kk.kernels()["prefix_attention_plan"](descs, nd, lanes, 3, groups, 1, 32, 4, 148, None, 4, C.byref(kk.PrefixPlan())) == kk.KK_EINVAL
    assert kk.kernels()["prefix_attention_plan"](descs, nd, lanes, 3, groups, 1, 32, 4, 148, None, 0, None) == kk.KK_EINVAL


def valid_desc(kk):
    d = kk.PrefixAttnDesc()
    d.pools = kk.KvPools(1 << 20, 1 << 21, 8, 4, 2, 4, 64, 8)
    d.layer, d.q_heads, d.scale = 1, 32, 0.125
    d.plan = kk.PrefixPlan(5, 4, 8, 3, 1, 9, 32, 4, 1000)
    d.descs = d.lanes = d.groups = d.items = 1 << 12
    d.query = d.output = d.workspace = 1 << 16
    d.query_stride = d.output_stride = 2048
    d.workspace_bytes = 264000
    return d


@pytest.mark.parametrize("change", [
    dict(layer=2), dict(q_heads=16), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(descs=None), dict(lanes=None), dict(groups=None), dict(items=None),
    dict(descs=(1 << 12) + 2), dict(lanes=(1 << 12) + 1), dict(groups=(1 << 12) + 2), dict(items=(1 << 12) + 2),
    dict(query=None), dict(output=None), dict(query=(1 << 16) + 8), dict(output=(1 << 16) + 2),
    dict(query_stride=2044), dict(output_stride=2040), dict(workspace=None), dict(workspace=(1 << 16) + 8),
    dict(workspace_bytes=263999), dict(pools=(1 << 20, 1 << 21, 8, 4, 2, 4, 128, 8)),
    dict(pools=(1 << 20, 1 << 21, 8, 4, 2, 4, 64, 12)), dict(pools=(1 << 20, 1 << 21, 8, 4, 2, 8, 64, 8)),
    dict(pools=((1 << 20) + 8, 1 << 21, 8, 4, 2, 4, 64, 8)), dict(plan=(5, 6, 8, 3, 1, 9, 32, 4, 1000)),
    dict(plan=(5, 4, 0, 3, 1, 9, 32, 4, 1000)), dict(plan=(5, 4, 8, 3, 1, 9, 32, 8, 1000)),
    dict(plan=(5, 4, 8, 3, 1, 9, 32, 4, 1 << 33)),
], ids=str)
def test_attention_refuses(kk, change):
    d = valid_desc(kk)
    for name, value in change.items():
        kind = {"pools": kk.KvPools, "plan": kk.PrefixPlan}.get(name)
        setattr(d, name, kind(*value) if kind else value)
    assert kk.kernels()["prefix_attention"](C.byref(d), None) == kk.KK_EINVAL


def test_attention_without_lanes_launches_nothing(kk):
    d = valid_desc(kk)
    d.plan = kk.PrefixPlan(0, 0, 8, 0, 0, 0, 32, 4, 0)
    assert kk.kernels()["prefix_attention"](C.byref(d), None) == 0
    assert kk.kernels()["prefix_attention"](None, None) == kk.KK_EINVAL


# ---- numerics (GPU) -----------------------------------------------------------


class Setup:
    """Pools filled for a list of tables; every byte no table covers is NaN."""

    def __init__(self, kk, tables, pages, hq, hkv, seed=0, sms=148, group=True, scale=0.125, layers=2, q_scale=1.5):
        self.kk, self.hq, self.hkv, self.layers, self.scale, self.tables = kk, hq, hkv, layers, scale, tables
        gen = torch.Generator(device="cuda").manual_seed(seed)
        nm, ne = max(1, pages.next[0]), pages.next[1]
        nan = float("nan")
        self.micro = torch.full((nm, layers, 2, pages.page, hkv, 64), nan, dtype=torch.half, device="cuda")
        self.extent = torch.full((max(1, ne), layers, 2, 64, hkv, 64), nan, dtype=torch.half, device="cuda")
        most = {}
        for t in tables:
            for slot, _, n, kind in t:
                most[(slot, kind)] = max(n, most.get((slot, kind), 0))
        for (slot, kind), n in most.items():
            pool = self.extent if kind else self.micro
            pool[slot, :, :, :n] = torch.randn(layers, 2, n, hkv, 64, generator=gen, device="cuda").half()
        self.pools = kk.KvPools(p(self.micro), p(self.extent) if ne else 0, nm, ne, layers, hkv, 64, pages.page)
        B = len(tables)
        self.q = (torch.randn(B, hq * 64 + 8, generator=gen, device="cuda") * q_scale).half()
        self.out = torch.full((B, hq * 64 + 16), 5.0, dtype=torch.half, device="cuda")
        descs, lanes, nd = pack(kk, tables)
        self.full = (descs, (kk.AttnLane * max(1, B))(*lanes), nd)
        groups, ng = find(kk, descs, lanes, B) if group else ((kk.PrefixGroup * 1)(), 0)
        rc, items, self.plan = plan_for(kk, descs, nd, lanes, B, groups, ng, hq, hkv, sms)
        assert rc == 0 and self.plan.num_items <= 65536
        self.ng, self.groups, self.items, self.lanes = ng, groups, items, lanes
        self.dev = [to_device_bytes(a) for a in (descs, lanes, groups, (kk.PrefixItem * max(1, self.plan.num_items))(
            *items[:self.plan.num_items]))]
        size = kk.kernels()["prefix_attention_workspace_bytes"](C.byref(self.plan))
        self.ws = torch.full((max(16, size),), 0xFF, dtype=torch.uint8, device="cuda")  # NaN
        d = self.desc = kk.PrefixAttnDesc()
        d.pools, d.q_heads, d.scale, d.plan = self.pools, hq, scale, self.plan
        d.descs, d.lanes, d.groups, d.items = map(p, self.dev)
        d.query, d.query_stride, d.output, d.output_stride = p(self.q), self.q.shape[1], p(self.out), self.out.shape[1]
        d.workspace, d.workspace_bytes = p(self.ws), size

    def run(self, layer=1, stream=None):
        self.desc.layer = layer
        rc = self.kk.kernels()["prefix_attention"](C.byref(self.desc), stream.cuda_stream if stream else None)
        assert rc == 0, rc

    def reference(self, layer, b):
        """64-bit result of lane b, and the size of the errors that FP32 sums leave in it."""
        parts = [(self.extent if k else self.micro)[s, layer, :, :n] for s, _, n, k in self.tables[b] if n]
        if not parts:
            return torch.zeros(self.hq, 64, dtype=torch.float64, device="cuda"), 0.0
        k, v = torch.cat(parts, 1).double()
        q = self.q[b, :self.hq * 64].double().view(self.hkv, -1, 64)
        score = torch.einsum("hgd,thd->hgt", q, k) * self.scale
        out = torch.einsum("hgt,thd->hgd", torch.softmax(score, -1), v).reshape(self.hq, 64)
        top = float(torch.einsum("hgd,thd->hgt", q.abs(), k.abs()).max()) * self.scale
        # A score is a sum of 64 products in FP32 (2^-23 a step at most): a weight is off by 2^-17 top
        # relative, and by 2^-21 for the exponential and its argument; a quotient of two such sums by
        # twice that. A weight of a shared token is rounded to FP16, off by 2^-11 at most. Sums over T
        # tokens add 2^-23 a token. All of it scales with the largest value.
        size = float(v.abs().max()) * (2 * (top * 2.0 ** -17 + 2.0 ** -21) + 2.0 ** -11 + (k.shape[0] + 64) * 2.0 ** -23)
        return out, size

    def check(self, layer=1):
        torch.cuda.synchronize()
        assert self.kk.kernels()["device_status"](None) == 0
        for b in range(len(self.tables)):
            ref, size = self.reference(layer, b)
            got = self.out[b, :self.hq * 64].double().view(self.hq, 64)
            bound = ref.abs() * 2.0 ** -11 + 2.0 ** -25 + size  # half an FP16 step, and the FP32 sums
            over = (got - ref).abs() - bound
            assert bool(torch.isfinite(got).all()), f"lane {b}"
            assert float(over.max()) <= 0, f"lane {b}: {float(over.max())} over {size}"
        assert bool((self.out[:, self.hq * 64:] == 5.0).all())


def forks(pages, prefix, tails, ragged=False, extents=True):
    shared = pages.table(prefix, ragged=ragged, extents=extents)
    return [shared + pages.table(n, prefix, ragged=ragged, extents=extents) for n in tails]


@gpu_test
@pytest.mark.parametrize("prefix", [1, 7, 8, 63, 64, 65, 127, 128, 129, 256, 500, 1023, 1500])
@pytest.mark.parametrize("sms", [1, 148])
def test_prefix_lengths(kk, prefix, sms):
    pages = Pages(random.Random(prefix))
    s = Setup(kk, forks(pages, prefix, [0, 1, 9, 70]), pages, 32, 4, prefix, sms)
    assert s.ng == 1
    for layer in (0, 1):
        s.run(layer)
        s.check(layer)


@gpu_test
@pytest.mark.parametrize("hkv,ratio", [(1, 1), (1, 16), (2, 3), (3, 8), (4, 7), (8, 4), (8, 1), (5, 12), (16, 2)])
@pytest.mark.parametrize("lanes", [2, 17, 40])
def test_prefix_head_layouts(kk, hkv, ratio, lanes):
    rng = random.Random(hkv * ratio + lanes)
    pages = Pages(rng)
    s = Setup(kk, forks(pages, 700, [rng.randint(0, 200) for _ in range(lanes)]), pages, hkv * ratio, hkv, lanes, rng.choice([5, 148]))
    s.run()
    s.check()


@gpu_test
@pytest.mark.parametrize("page", [8, 16, 32, 64])
@pytest.mark.parametrize("extents", [True, False])
def test_prefix_pages_partly_filled(kk, page, extents):
    """Pages that end anywhere inside a tile; what stands behind their valid tokens is NaN."""
    rng = random.Random(page)
    pages = Pages(rng, page)
    tables = forks(pages, 1100, [0, 3, 100, 400], True, extents) + forks(pages, 333, [65, 0], True, extents)
    tables += [pages.table(50, ragged=True), []]
    for sms in (2, 148):
        s = Setup(kk, tables, pages, 16, 2, page, sms)
        assert s.ng == 2
        s.run()
        s.check()


@gpu_test
def test_prefix_many_groups_and_lanes_without_one(kk):
    rng = random.Random(5)
    pages = Pages(rng)
    tables = []
    for n in (2, 33, 1, 5, 130):
        tables += forks(pages, rng.randint(64, 900), [rng.choice([0, 1, 8, 40, 300]) for _ in range(n)])
    tables += [[], [], pages.table(1)]
    s = Setup(kk, tables, pages, 32, 4, 6)
    assert s.ng == 4
    s.run()
    s.check()
    alone = Setup(kk, tables, pages, 32, 4, 6, group=False)  # every lane by itself: the same results
    assert alone.plan.num_shared == 0
    alone.run()
    alone.check()


@gpu_test
@pytest.mark.parametrize("score", [6.0, 9.0, 10.5, 11.0, 12.0, 13.0, 14.0])
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
def test_prefix_one_token_outweighs_the_rest(kk, score, group):
    """A first token with a score far above all others' (which are 0) and no value of its own: what is left
    of the result are the others' weights, e^-score each, and rounds no worse than any weight does."""
    pages = Pages(random.Random(21))
    tables = forks(pages, 4000, [0, 0])
    s = Setup(kk, tables, pages, 8, 1, 22, sms=1, group=group)  # few parts: many of the others stand next to it
    for pool in (s.micro, s.extent):
        for part, value in ((0, 0.0), (1, 1.0)):
            x = pool[:, :, part]
            x[~torch.isnan(x)] = value
    slot, _, _, kind = tables[0][0]
    first = (s.extent if kind else s.micro)[slot, :, :, 0]
    first.zero_()
    first[:, 0, :, 0] = score / s.scale
    s.q.zero_()
    s.q.view(2, -1)[:, :512:64] = 1.0
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    rest = 3999 * torch.exp(torch.tensor(-score, dtype=torch.float64))
    want = float(rest / (1 + rest))
    error = (s.out[:, :512].double() / want - 1).abs().max()
    # A weight and the result in FP16, half a step each; exponentials, their argument (off by 2^-24 of 21) and
    # FP32 sums of 4,000 terms in order: 2^-16.
    assert float(error) <= 2 * 2.0 ** -11 + 2.0 ** -22 + 2.0 ** -16


@gpu_test
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("token", [0, 77, 149, 160])
def test_prefix_infinities_and_nan_among_the_keys(kk, group, value, token):
    """One coordinate of one key: a score of +inf or NaN makes the row NaN, one of -inf weighs nothing; other KV
    heads, and lanes that do not see the token, are as they would be."""
    pages = Pages(random.Random(23))
    tables = forks(pages, 150, [30, 0, 12])
    s = Setup(kk, tables, pages, 12, 2, 24, group=group)
    at = 0
    for slot, _, n, kind in tables[0]:
        if at <= token < at + n:
            (s.extent if kind else s.micro)[slot, 1, 0, token - at, 1, 5] = value
        at += n
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    seen = 0
    for b in range(3):
        ref, _ = s.reference(1, b)
        got = s.out[b, :12 * 64].double().view(12, 64)
        lost = torch.isnan(ref)
        seen += int(lost.sum())
        assert bool((torch.isnan(got) == lost).all())
        assert not bool(lost[:6].any())
        # As in `reference`, with 2^8 for the largest sum of a score's terms (about 20 here; the rest leaves room
        # for the FP32 sums) and 8 for the largest value.
        over = (got - ref).abs() - (ref.abs() * 2.0 ** -11 + 2.0 ** -25 + 8 * (2.0 ** -8 + 2.0 ** -11))
        assert float(over[~lost].max()) <= 0
    assert seen > 0


@gpu_test
def test_prefix_pages_without_tokens(kk):
    """Tables with pages that hold nothing yet, more in a row than a warp looks at once, at the start, inside and
    at the end; lanes and prefixes made of nothing else."""
    pages = Pages(random.Random(17))

    def empty(n):
        return [(pages.take(0), 0, 0, 0) for _ in range(n)]

    shared = empty(1) + pages.table(100) + empty(70) + pages.table(200, 100) + empty(33)
    tables = [shared + tail for tail in (empty(40) + pages.table(30) + empty(1), [], empty(3), pages.table(5) + empty(65))]
    nothing = empty(2)
    tables += [nothing + pages.table(9), list(nothing), empty(1), []]
    for sms in (1, 148):
        s = Setup(kk, tables, pages, 8, 2, 18, sms)
        assert s.ng == 1
        s.run()
        s.check()


@gpu_test
def test_prefix_long_runs_and_growing_maxima(kk):
    """Hundreds of tiles per block, scores that grow along the context (the running maximum moves again
    and again) and lie far apart."""
    pages = Pages(random.Random(8))
    s = Setup(kk, forks(pages, 20000, [5, 0, 33]), pages, 8, 1, 9, sms=2, q_scale=4.0)
    ramp = 1.0 + 4.0 * torch.arange(max(1, pages.next[1]), device="cuda").half() / pages.next[1]
    s.extent[:, :, 0] *= ramp[:, None, None, None, None]
    s.run()
    s.check()
    s.micro.abs_()
    s.extent.abs_()
    s.q.neg_().abs_().neg_()  # every score negative and large
    s.run()
    s.check()


@gpu_test
def test_prefix_chunk_positions_share_pages(kk):
    """The positions of a prompt chunk: lane i sees the prefix and the chunk's first i + 1 tokens, which
    stand in the same pages for every lane."""
    pages = Pages(random.Random(10), 16)
    shared, chunk = pages.table(1000), pages.table(64)
    tables = []
    for i in range(64):
        own = [e for e in chunk if e[1] <= i]
        slot, begin, _, kind = own[-1]
        tables.append(shared + [(s_, b + 1000, n, k_) for s_, b, n, k_ in own[:-1]] + [(slot, begin + 1000, i + 1 - begin, kind)])
    s = Setup(kk, tables, pages, 32, 4, 11)
    assert s.ng == 1 and s.groups[0].token_count == 1000
    s.run()
    s.check()


@gpu_test
@pytest.mark.parametrize("page", [8, 64])
def test_prefix_pages_behind_32_bit_offsets(kk, page):
    """Pages that begin more than 2^32 elements behind the pool's start (an 8.6 GB pool)."""
    pages = Pages(random.Random(19), page)
    pages.next = [0, 16400] if page == 8 else [16400, 0]
    s = Setup(kk, forks(pages, 300, [20, 0, 70]), pages, 32, 16, 20)
    assert (s.extent if page == 8 else s.micro)[16400:].data_ptr() - p(s.extent if page == 8 else s.micro) > 2 ** 33
    s.run()
    s.check()


@gpu_test
def test_prefix_matches_per_lane_attention(kk):
    K = kk.kernels()
    pages = Pages(random.Random(12))
    s = Setup(kk, forks(pages, 1777, [0, 12, 260, 64, 1]), pages, 32, 4, 13)
    s.run()
    descs, lanes, nd = s.full
    items = (kk.AttnItem * 4096)()
    n = K["attention_plan_balanced"](descs, lanes, 5, 20, items, 4096)
    dev = [to_device_bytes(a) for a in (descs, lanes, items)]
    size = K["attention_workspace_bytes"](5, n, 32, 64)
    ws = torch.zeros(size, dtype=torch.uint8, device="cuda")
    out = torch.zeros(5, 2048, dtype=torch.half, device="cuda")
    rc = K["paged_decode_attention"](C.byref(s.pools), 1, 32, p(dev[0]), p(dev[1]), 5, p(dev[2]), n, p(s.q), s.q.shape[1],
                                     p(out), 2048, s.scale, p(ws), size, None)
    assert rc == 0
    s.check()
    for b in range(5):
        ref, size = s.reference(1, b)
        # Both lie within half an FP16 step and their FP32 sums of the same value.
        bound = 2 * (ref.abs() * 2.0 ** -11 + 2.0 ** -25 + size)
        got = out[b].double() - s.out[b, :2048].double()
        assert bool((got.view(32, 64).abs() <= bound).all())


@gpu_test
def test_prefix_streams_capture_and_workspace(kk):
    """Two calls on two streams with a workspace each; captured calls that share one workspace in turn; the
    same inputs give the same bits."""
    rng = random.Random(14)
    sets = []
    for seed in (1, 2):
        pages = Pages(rng)
        sets.append(Setup(kk, forks(pages, 900, [3, 50, 0, 17, 128]), pages, 32, 4, seed))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for s, stream in zip(sets, streams):
            s.run(stream=stream)
    for s in sets:
        s.check()
    first = [s.out.clone() for s in sets]
    if sets[0].ws.numel() < sets[1].ws.numel():
        sets.reverse()
        first.reverse()
    sets[1].desc.workspace = p(sets[0].ws)
    torch.cuda.synchronize()
    graphs = []
    for s in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run(stream=torch.cuda.current_stream())
        graphs.append(g)
    for _ in range(3):
        for s in sets:
            s.out[:, :2048].zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s, want in zip(sets, first):
            assert torch.equal(s.out, want)
    for g, s in zip(graphs, sets):  # new values behind the same plan
        s.q.normal_()
        g.replay()
        s.check()


@gpu_test
def test_prefix_reports_bad_pages_and_items(kk):
    K = kk.kernels()
    pages = Pages(random.Random(15))
    tables = forks(pages, 300, [20, 5])
    s = Setup(kk, tables, pages, 8, 2, 16)
    s.run()
    s.check()
    good = s.out.clone()
    descs, lanes, nd = s.full
    # A page outside its pool, one over its capacity, an unknown kind: left out and reported.
    for at in (0, len(tables[0]) - 1):
        for change in (dict(slot=1 << 20), dict(valid_tokens=65), dict(kind=7)):
            bad = (kk.PageDesc * nd)(*descs[:nd])
            for name, value in change.items():
                setattr(bad[at], name, value)
            dev = to_device_bytes(bad)
            s.desc.descs = p(dev)
            s.run()
            torch.cuda.synchronize()
            assert K["device_status"](None) == 2
            keep, s.tables = s.tables, [list(t) for t in tables]
            for t in s.tables:
                if t[at:at + 1] == tables[0][at:at + 1]:
                    del t[at]
            s.check()
            s.tables = keep
    s.desc.descs = p(s.dev[0])
    # Items that do not fit the plan are reported and write nothing outside the workspace.
    n = s.plan.num_items
    for at, change in ((0, dict(owner=9)), (0, dict(kv_head=2)), (0, dict(desc_end=nd + 1)), (0, dict(part_row=(1 << 32) - 1)),
                       (0, dict(row_tile=5)), (0, dict(row_tiles=3)), (0, dict(token_tiles=0)), (n - 1, dict(owner=2)),
                       (0, dict(lane_count=3)), (0, dict(lane_begin=1 << 31)), (n - 1, dict(part_row=s.plan.part_rows - 3)), (n - 1, dict(desc_begin=nd, desc_end=nd - 1)), (n - 1, dict(row_tiles=1))):
        items = (kk.PrefixItem * n)(*s.items[:n])
        for name, value in change.items():
            setattr(items[at], name, value)
        dev = to_device_bytes(items)
        s.desc.items = p(dev)
        s.run()
        torch.cuda.synchronize()
        assert K["device_status"](None) == 3, change
    # More pages than the item's tiles: the rest is left out and reported.
    items = (kk.PrefixItem * n)(*s.items[:n])
    items[0].token_tiles, items[0].desc_begin, items[0].desc_end = 1, 0, len(tables[0])
    dev = to_device_bytes(items)
    s.desc.items = p(dev)
    s.run()
    torch.cuda.synchronize()
    assert K["device_status"](None) == 3
    s.desc.items = p(s.dev[3])
    s.run()
    s.check()
    assert torch.equal(s.out, good)


@gpu_test
@pytest.mark.parametrize("score", [1.25, 1.375, 2.75, 3.25, 5.5, 6.375, 6.875])
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
def test_prefix_weights_keep_more_bits_than_the_result(kk, score, group):
    """All tokens but the first have the same score and value, so that their weights round alike; the value puts
    the result right below 1, where half an FP16 step is 2^-12 of it. A weight of FP16's 11 bits (off by 2^-12.2
    to 2^-11.1 at these scores) does not do."""
    tokens = 1000
    pages = Pages(random.Random(25))
    s = Setup(kk, forks(pages, tokens, [0, 0]), pages, 8, 1, 26, sms=1, group=group)
    for pool in (s.micro, s.extent):
        for part in (0, 1):
            x = pool[:, :, part]
            x[~torch.isnan(x)] = 0.0
    rest = (tokens - 1) * torch.exp(torch.tensor(-score, dtype=torch.float64))
    share = float(rest / (1 + rest))
    value = torch.tensor(1 / share).half()
    while float(value) * share >= 1:
        value = torch.nextafter(value, torch.zeros_like(value))
    want = float(value) * share
    assert 0.99 < want < 1
    for pool in (s.micro, s.extent):
        x = pool[:, :, 1]
        x[~torch.isnan(x)] = float(value)
    slot, _, _, kind = s.tables[0][0]
    first = (s.extent if kind else s.micro)[slot, :, :, 0]
    first.zero_()
    first[:, 0, :, 0] = score / s.scale
    s.q.zero_()
    s.q.view(2, -1)[:, :512:64] = 1.0
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    # Half a step of the result. Weights: 2^-18.5 each in the products and in the sum, their argument (7 + 16 at
    # most in size, off by 2^-24 of that), 22 bits of them in the products. FP32 sums: two products for each of
    # 63 steps of 16 tokens, 2^-23 a step; fewer additions in the sum of the weights.
    bound = 2.0 ** -12 + 2 * 2.0 ** -18.5 + 2 * 2.0 ** -19.4 + 2.0 ** -21 + 2 * 63 * 2.0 ** -23 + 64 * 2.0 ** -24
    assert float((s.out[:, :512].double() - want).abs().max()) <= bound


@gpu_test
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
@pytest.mark.parametrize("page,prefix", [(8, 1), (8, 64), (8, 1333), (16, 700), (64, 3001), (8, 9000)])
def test_prefix_every_token_counts_once(kk, group, page, prefix):
    """Equal scores, and a value of one in dim t % 64 of token t: a dim of the result is the share of its tokens.
    A token too few or too many moves one by 64 / tokens of itself, 2^-7.2 or more."""
    rng = random.Random(page + prefix)
    pages = Pages(rng, page)
    tables = forks(pages, prefix, [0, 1, 77, 300], ragged=True)
    s = Setup(kk, tables, pages, 16, 2, 27, group=group)
    eye = torch.eye(64, dtype=torch.half, device="cuda")
    for t in tables:
        at = 0
        for slot, _, n, kind in t:
            ids = torch.arange(at, at + n, device="cuda") % 64
            (s.extent if kind else s.micro)[slot, :, 1, :n] = eye[ids][None, :, None, :]
            at += n
    s.q.zero_()
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    for b, t in enumerate(tables):
        tokens = sum(e[2] for e in t)
        want = torch.tensor([(tokens + 63 - d) // 64 for d in range(64)], dtype=torch.float64, device="cuda") / tokens
        # Half an FP16 step; weights, in the products and in their sum; FP32 sums, 2^-24 a token: 2^-9.8 at most.
        bound = want * (2.0 ** -11 + 2 * 2.0 ** -18.5 + tokens * 2.0 ** -24) + 2.0 ** -25
        over = (s.out[b, :1024].double().view(16, 64) - want).abs() - bound
        assert float(over.max()) <= 0


@gpu_test
@pytest.mark.parametrize("score", [0.0, 0.25, 0.6, -1.1])
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
def test_prefix_equal_scores_have_equal_weights(kk, score, group):
    """A value of +1000 is met by one of -1000 with the same score, wherever the two stand in a tile:
    nothing is left of the sums but what the weights differ by."""
    tokens = 1536
    pages = Pages(random.Random(28))
    s = Setup(kk, forks(pages, tokens, [0, 0]), pages, 8, 1, 29, sms=3, group=group)
    at = 0
    for slot, _, n, kind in s.tables[0]:
        page = (s.extent if kind else s.micro)[slot]
        t = torch.arange(at, at + n, device="cuda")
        page[:, 0, :n] = 0.0
        page[:, 0, :n, :, 0] = score / s.scale
        page[:, 1, :n] = 0.0
        for dim in range(64):  # +1000 for tokens t % 8 == a, -1000 for t % 8 == b
            a, b = dim % 8, dim // 8
            if a != b:
                page[:, 1, :n, :, dim] = (1000.0 * ((t % 8 == a).half() - (t % 8 == b).half()))[None, :, None]
        at += n
    # One token outweighs them, so that their weights are no powers of two; it has no value.
    slot, _, _, kind = s.tables[0][0]
    first = (s.extent if kind else s.micro)[slot, :, :, :8]
    first.zero_()
    first[:, 0, 0, :, 0] = 2.0 / s.scale
    s.q.zero_()
    s.q.view(2, -1)[:, :512:64] = 1.0
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    # A weight is off by 2^-21 at most, an eighth of the tokens have it, and half an FP16 step of what is left.
    assert float(s.out[:, :512].abs().max()) <= 2 * 125 * 2.0 ** -21 * (1 + 2.0 ** -10)


@gpu_test
def test_prefix_lanes_that_do_not_fit_the_plan(kk):
    """Lanes whose partial rows lie outside the plan's are reported and their rows left as they were; the calls
    behind, which use the same workspace, are not touched by them."""
    pages = Pages(random.Random(32))
    tables = forks(pages, 3000, [20, 500, 64, 7])
    s = Setup(kk, tables, pages, 32, 4, 33)
    s.run()
    s.check()
    good = s.out.clone()
    lanes = (kk.AttnLane * 4)(*s.lanes[:4])
    for b in range(4):
        lanes[b].item_offset = 0xFFFFFFF0
    dev = to_device_bytes(lanes)
    for b in range(4):
        lanes[b].item_offset, lanes[b].item_count = s.lanes[b].item_offset, 0xFFFFFFFF
    more = to_device_bytes(lanes)
    for bad in (dev, more):
        s.out[:, :2048] = 3.0
        s.desc.lanes = p(bad)
        s.run()
        torch.cuda.synchronize()
        assert kk.kernels()["device_status"](None) == 3
        assert bool((s.out[:, :2048] == 3.0).all())
        for _ in range(5):
            s.desc.lanes = p(bad)
            s.run()
            s.desc.lanes = p(s.dev[1])
            s.run()
        torch.cuda.synchronize()
        assert kk.kernels()["device_status"](None) == 3
        assert torch.equal(s.out, good)


@gpu_test
@pytest.mark.parametrize("group", [True, False], ids=["shared", "own"])
@pytest.mark.parametrize("size", [30.0, 300.0, 1000.0, 4000.0, 10000.0, 20000.0])
def test_prefix_scores_of_any_size(kk, group, size):
    """Scores up to 10^10, where FP32 tells neighbours further apart than FP16's whole range of weights: a row's
    result is the value of its highest token, wherever that one leads by more than the scores are off."""
    pages = Pages(random.Random(35))
    s = Setup(kk, forks(pages, 1500, [0, 40, 300]), pages, 8, 2, 36, sms=3, group=group, q_scale=size)
    for pool in (s.micro, s.extent):
        pool[:, :, 0] *= min(size, 10000.0)
    s.q.clamp_(-60000.0, 60000.0)
    s.run()
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    told = 0
    for b, t in enumerate(s.tables):
        k, v = torch.cat([(s.extent if kind else s.micro)[slot, 1, :, :n] for slot, _, n, kind in t], 1).double()
        q = s.q[b, :512].double().view(2, -1, 64)
        score = torch.einsum("hgd,thd->hgt", q, k) * s.scale
        top, at = score.topk(2, -1)
        terms = torch.einsum("hgd,thd->hgt", q.abs(), k.abs()).amax(-1) * s.scale
        # 64 products in FP32, 2^-23 a step at most; as much again for the factor and the maximum. A lead of 40 more
        # leaves e^-40 of the others.
        lead = top[..., 0] - top[..., 1] > 40 + 2 * 2.0 ** -17 * terms
        want = v[at[..., 0], torch.arange(2, device="cuda")[:, None]]  # [head, query head, 64]
        got = s.out[b, :512].double().view(2, -1, 64)
        assert bool(torch.isfinite(got).all()), f"lane {b}"
        assert bool(((got - want).abs() <= want.abs() * 2.0 ** -11 + 2.0 ** -25)[lead].all()), f"lane {b}"
        told += int(lead.sum())
    assert told >= 12  # of 24


@gpu_test
def test_prefix_lanes_without_any_tokens(kk):
    """Nothing to plan: the rows are zeros."""
    pages = Pages(random.Random(37))
    s = Setup(kk, [[], [], []], pages, 32, 4, 38)
    assert s.plan.num_items == 0
    s.run()
    s.check()


@gpu_test
@pytest.mark.parametrize("groups,lanes,prefix,own,hq,hkv", [
    (40, 3, 300, 200, 32, 8),     # more prefixes times KV heads than SMs: rounds of blocks
    (19, 2, 64, 1000, 8, 8),
    (1, 600, 200, 20, 16, 1),     # 75 tiles of query rows over one prefix
    (1, 700, 130, 9, 28, 4),
])
def test_prefix_many_groups_and_many_rows(kk, groups, lanes, prefix, own, hq, hkv):
    rng = random.Random(groups + lanes)
    pages = Pages(rng)
    tables = []
    for _ in range(groups):
        tables += forks(pages, prefix, [rng.randint(0, own) for _ in range(lanes)])
    s = Setup(kk, tables, pages, hq, hkv, 39)
    assert s.ng == groups
    s.run()
    s.check()


@gpu_test
def test_prefix_short_lanes_among_long_ones(kk):
    """Lanes that share more with some neighbours than with others, in every order."""
    rng = random.Random(40)
    pages = Pages(rng)
    a, b, c = pages.table(64), pages.table(2000, 64), pages.table(500, 64)
    tables = []
    for kind in "saabbsacasbb":
        head = {"s": a, "a": a + b, "b": a + c, "c": a + b + c}[kind]
        tables.append(head + pages.table(rng.choice([0, 1, 40]), sum(e[2] for e in head)))
    s = Setup(kk, tables, pages, 32, 4, 41)
    assert s.ng >= 1
    s.run()
    s.check()
