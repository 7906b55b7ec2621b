"""kk_kv_append_rope: rotating KV append of ragged batches. The refusals run on
the CPU (nothing is launched); the numerics run on the GPU against an 80-bit
host reference."""
import ctypes as C

import numpy as np
import pytest
import torch

from gpu_util import p, to_device_bytes

HAVE_GPU = torch.cuda.is_available()
gpu = [pytest.mark.gpu, pytest.mark.skipif(not HAVE_GPU, reason="needs a CUDA device")]


def gpu_test(fn):
    for mark in gpu:
        fn = mark(fn)
    return fn


# ---- refusals (CPU) ---------------------------------------------------------


def valid_desc(kk):
    d = kk.KvAppendDesc()
    d.pools = kk.KvPools(1 << 20, 1 << 21, 8, 4, 2, 2, 64, 8)
    d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 1, 3, 4, 64, 10000.0
    d.slots = d.positions = 1 << 12
    d.query = d.key = d.value = d.query_out = 1 << 16
    d.query_stride = d.query_out_stride = 256
    d.key_stride = d.value_stride = 128
    return d


@pytest.mark.parametrize("change", [
    dict(layer=2), dict(rotary_dim=24), dict(rotary_dim=80), dict(theta=0.0), dict(theta=0.5),
    dict(theta=float("nan")), dict(theta=float("inf")), dict(slots=None), dict(positions=None),
    dict(query=None), dict(query_out=None), dict(key=None), dict(value=None), dict(key=(1 << 16) + 2),
    dict(query=(1 << 16) + 8), dict(value_stride=132), dict(key_stride=120), dict(query_stride=248),
    dict(query_out_stride=248), dict(query_stride=264), dict(cos_sin=1 << 14),  # no table_positions
    dict(slots=(1 << 12) + 2), dict(positions=(1 << 12) + 1),
    dict(cos_sin=(1 << 14) + 4, table_positions=9), dict(q_heads=1 << 20),
    dict(pools=(1 << 20, 1 << 21, 8, 4, 2, 2, 60, 8)), dict(pools=(1 << 20, 1 << 21, 8, 4, 0, 2, 64, 8)),
    dict(pools=(1 << 20, 1 << 21, 8, 4, 2, 2, 64, 24)), dict(pools=((1 << 20) + 4, 1 << 21, 8, 4, 2, 2, 64, 8)),
])
def test_append_refuses(kk, change):
    d = valid_desc(kk)
    for name, value in change.items():
        setattr(d, name, kk.KvPools(*value) if name == "pools" else value)
    assert kk.kernels()["kv_append_rope"](C.byref(d), None) == kk.KK_EINVAL


def test_append_without_rows_launches_nothing(kk):
    d = valid_desc(kk)
    d.rows = 0
    assert kk.kernels()["kv_append_rope"](C.byref(d), None) == 0
    assert kk.kernels()["kv_append_rope"](None, None) == kk.KK_EINVAL


# ---- numerics (GPU) ---------------------------------------------------------


def rotate_ref(x, positions, rotary, theta, table=None):
    """x [rows, heads, dim] -> rotated, in 80-bit arithmetic."""
    x = x.astype(np.longdouble)
    half = rotary // 2
    if table is None:
        power = np.arange(half, dtype=np.longdouble) * 2 / np.longdouble(max(rotary, 1))
        angle = positions.astype(np.longdouble)[:, None] / np.power(np.longdouble(theta), power)
        cos, sin = np.cos(angle), np.sin(angle)
    else:
        cos, sin = (table[positions, :, i].astype(np.longdouble) for i in (0, 1))
    a, b = x[..., :half].copy(), x[..., half:rotary].copy()
    x[..., :half] = a * cos[:, None] - b * sin[:, None]
    x[..., half:rotary] = b * cos[:, None] + a * sin[:, None]
    return x


def assert_rounded(got, ref, size):
    """FP16 results of FP32 sums of two products: half an FP16 step of the value
    (2^-11, or 2^-25 among the subnormals), and of size = |a| + |b|: 2^-22 for
    the products, their sum and cos / sin's own roundings (four of 2^-24), and
    2^-17.9 for an angle off by 4e-6 rad at the farthest position."""
    err = np.abs(got.astype(np.longdouble) - ref)
    bound = np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 + size * (2.0 ** -22 + 4e-6)
    assert (err <= bound).all(), float((err - bound).max())


CASES = [
    # rows, q_heads, kv_heads, dim, rotary, page, extents, far
    (1, 32, 4, 64, 64, 8, True, 2048),
    (5, 8, 2, 64, 64, 8, True, 100),
    (64, 32, 4, 64, 32, 16, False, 4096),
    (1, 1, 1, 8, 0, 8, True, 5),
    (7, 3, 3, 16, 16, 8, False, 1 << 20),
    (129, 7, 1, 128, 128, 64, False, 1 << 31),
    (33, 0, 8, 128, 64, 8, True, 1000),
    (3, 5, 1, 256, 256, 32, False, 1 << 32),
    (2, 2, 2, 320, 256, 8, True, 70),
    (1025, 6, 2, 64, 48, 8, True, 8192),
    (1500, 32, 8, 128, 128, 8, True, 1 << 20),
    # Rows per thread block: one wave of blocks holds 740, 5,920 at most.
    (740, 2, 1, 16, 16, 8, True, 100),
    (741, 2, 1, 32, 16, 8, True, 100),
    (4999, 4, 2, 128, 64, 16, False, 100000),
    (5920, 2, 1, 16, 16, 8, True, 100),
    (5921, 3, 1, 24, 16, 8, True, 100),
]


def run_case(kk, rows, hq, hkv, dim, rotary, page, extents, far, seed=0, table=False, in_place=False,
             inactive=0.2, pad=0, stream=None):
    rng = np.random.RandomState(seed + rows)
    layers, layer = 3, 1
    micro_cap, extent_cap = rows // page + 3, (rows // 64 + 2 if extents else 0)
    shape = (layers, 2, page, hkv, dim)
    micro = torch.randn(micro_cap, *shape).half().cuda()
    extent = torch.randn(max(extent_cap, 1), layers, 2, 64, hkv, dim).half().cuda()
    pools = kk.KvPools(p(micro), p(extent) if extents else 0, micro_cap, extent_cap, layers, hkv, dim, page)
    places = [(0, s, t) for s in range(micro_cap) for t in range(page)]
    places += [(1, s, t) for s in range(extent_cap) for t in range(64)]
    rng.shuffle(places)
    places = places[:rows]
    active = rng.rand(rows) >= inactive
    active[0] = True
    slots = (kk.KvSlot * rows)(*[kk.KvSlot(s, t, k, int(a)) for (k, s, t), a in zip(places, active)])
    positions = rng.randint(0, far, rows, dtype=np.uint64).astype(np.uint32)
    positions[-1] = far - 1
    q = (rng.randn(rows, hq * dim + pad) * 2).astype(np.float16)
    k = (rng.randn(rows, hkv * dim + pad) * 2).astype(np.float16)
    v = (rng.randn(rows, hkv * dim + pad) * 2).astype(np.float16)
    # Padded rows may hold anything.
    q[~active], k[~active], v[~active] = np.nan, np.inf, np.nan
    dq, dk, dv = (torch.from_numpy(t).cuda() for t in (q, k, v))
    out = dq if in_place else torch.full_like(dq, 7.0)
    before_out, before_micro, before_extent = (t.clone() for t in (out, micro, extent))
    d = kk.KvAppendDesc()
    d.pools, d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = pools, layer, rows, hq, rotary, 10000.0
    d_slots, d_pos = to_device_bytes(slots), torch.from_numpy(positions.view(np.int32)).cuda()
    d.slots, d.positions = p(d_slots), p(d_pos)
    d.query, d.key, d.value, d.query_out = (p(t) if t.numel() else None for t in (dq, dk, dv, out))
    d.query_stride = d.query_out_stride = hq * dim + pad
    d.key_stride = d.value_stride = hkv * dim + pad
    cs = None
    if table:
        cs = rng.uniform(-1, 1, (far, rotary // 2, 2)).astype(np.float32)
        d_cs = torch.from_numpy(cs).cuda()
        d.cos_sin, d.table_positions, d.theta = p(d_cs), far, 0.0
    torch.cuda.synchronize()
    rc = kk.kernels()["kv_append_rope"](C.byref(d), stream.cuda_stream if stream else None)
    assert rc == 0
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0

    half = rotary // 2

    def size(x):
        s = np.zeros(x.shape)
        ab = np.abs(x[..., :half].astype(float)) + np.abs(x[..., half:rotary].astype(float))
        s[..., :half] = s[..., half:rotary] = ab
        return s

    def check(got, x, heads):
        x = x[:, :heads * dim].reshape(-1, heads, dim)
        got = got.reshape(x.shape)
        assert_rounded(got, rotate_ref(x, positions[active], rotary, 10000.0, cs), size(x))
        assert np.array_equal(got[..., rotary:], x[..., rotary:])  # copied dims

    if hq:
        got = out.cpu().numpy()
        check(got[active][:, :hq * dim], q[active], hq)
        keep = before_out.cpu().numpy()
        assert np.array_equal(got[~active], keep[~active], equal_nan=True)
        assert np.array_equal(got[:, hq * dim:], keep[:, hq * dim:], equal_nan=True)  # between the rows
    want = {0: before_micro, 1: before_extent}
    have = {0: micro, 1: extent}
    live = [pl for pl, a in zip(places, active) if a]
    keys = np.stack([have[kd][s, layer, 0, t].cpu().numpy() for kd, s, t in live]) if rows <= 200 else None
    if keys is None:
        idx = [(torch.tensor([s for kd, s, t in live if kd == w]).cuda(), torch.tensor([t for kd, s, t in live if kd == w]).cuda())
               for w in (0, 1)]
        sel = [np.array([i for i, (kd, _, _) in enumerate(live) if kd == w], int) for w in (0, 1)]
        keys, vals = np.zeros((len(live), hkv, dim), np.float16), np.zeros((len(live), hkv, dim), np.float16)
        for w in (0, 1):
            if len(sel[w]):
                keys[sel[w]] = have[w][idx[w][0], layer, 0, idx[w][1]].cpu().numpy()
                vals[sel[w]] = have[w][idx[w][0], layer, 1, idx[w][1]].cpu().numpy()
                for comp in (0, 1):
                    want[w][idx[w][0], layer, comp, idx[w][1]] = have[w][idx[w][0], layer, comp, idx[w][1]]
    else:
        vals = np.stack([have[kd][s, layer, 1, t].cpu().numpy() for kd, s, t in live])
        for kd, s, t in live:
            want[kd][s, layer, :, t] = have[kd][s, layer, :, t]
    check(keys, k[active], hkv)
    assert np.array_equal(vals.reshape(len(live), -1), v[active][:, :hkv * dim])
    # Nothing else of either pool changed.
    assert torch.equal(micro.view(torch.int16), want[0].view(torch.int16))
    assert torch.equal(extent.view(torch.int16), want[1].view(torch.int16))


@gpu_test
@pytest.mark.parametrize("case", CASES, ids=str)
def test_append_matches_reference(kk, case):
    run_case(kk, *case)


@gpu_test
@pytest.mark.parametrize("kw", [dict(table=True), dict(in_place=True), dict(pad=24), dict(inactive=1.0),
                                dict(in_place=True, pad=8, table=True)], ids=str)
@pytest.mark.parametrize("rows", [3, 1100])
def test_append_forms(kk, kw, rows):
    run_case(kk, rows, 8, 2, 64, 64, 8, True, 600, **kw)


@gpu_test
def test_append_on_another_stream_and_captured(kk):
    side = torch.cuda.Stream()
    run_case(kk, 70, 8, 2, 64, 64, 8, True, 600, stream=side)
    # Captured and replayed: the graph reads the arrays anew.
    rows, D = 9, 64
    micro = torch.zeros(4, 1, 2, 8, 1, D, dtype=torch.half, device="cuda")
    slots = (kk.KvSlot * rows)(*[kk.KvSlot(r // 8, r % 8, 0, 1) for r in range(rows)])
    d_slots = to_device_bytes(slots)
    pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
    x = torch.randn(rows, 3 * D, device="cuda").half()
    out = torch.zeros(rows, D, dtype=torch.half, device="cuda")
    d = kk.KvAppendDesc()
    d.pools = kk.KvPools(p(micro), 0, 4, 0, 1, 1, D, 8)
    d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 0, rows, 1, D, 10000.0
    d.slots, d.positions, d.query, d.key, d.value = p(d_slots), p(pos), p(x), p(x) + 2 * D, p(x) + 4 * D
    d.query_stride = d.key_stride = d.value_stride = 3 * D
    d.query_out, d.query_out_stride = p(out), D
    call = kk.kernels()["kv_append_rope"]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call(C.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    for step in (0, 5, 1000):
        pos.fill_(step)
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        xs = x.cpu().numpy().reshape(rows, 3, D)
        positions = np.full(rows, step, np.uint32)
        ab = np.abs(xs[..., :32].astype(float)) + np.abs(xs[..., 32:].astype(float))
        size = np.concatenate([ab, ab], -1)
        ref = rotate_ref(xs[:, :2], positions, D, 10000.0)
        assert_rounded(out.cpu().numpy(), ref[:, 0], size[:, 0])
        pages = micro.cpu().numpy()[:2, 0].transpose(1, 0, 2, 3, 4).reshape(2, 16, D)[:, :rows]
        assert_rounded(pages[0], ref[:, 1], size[:, 1])
        assert np.array_equal(pages[1], xs[:, 2])


@gpu_test
def test_append_reports_bad_rows_and_leaves_them(kk):
    """A slot outside its pool, a token outside its page, an unknown page kind
    and a position outside the table: the row is skipped and reported."""
    D, table = 64, 10
    slots = [kk.KvSlot(0, 0, 0, 1), kk.KvSlot(4, 1, 0, 1), kk.KvSlot(1, 8, 0, 1), kk.KvSlot(0, 1, 1, 1),
             kk.KvSlot(0, 2, 2, 1), kk.KvSlot(2, 3, 0, 1), kk.KvSlot(3, 3, 0, 1)]
    rows = len(slots)
    pos = torch.tensor([1, 1, 1, 1, 1, table, 9], dtype=torch.int32).cuda()
    codes = {0: 0, 1: 2, 2: 2, 3: 2, 4: 2, 5: 3, 6: 0}
    for bad in range(rows):
        micro = torch.zeros(4, 1, 2, 8, 1, D, dtype=torch.half, device="cuda")
        x = torch.randn(1, 3 * D, device="cuda").half()
        out = torch.full((1, D), 3.0, dtype=torch.half, device="cuda")
        cs = torch.tensor([1.0, 0.0], device="cuda").repeat(table, D // 2, 1)
        one = to_device_bytes((kk.KvSlot * 1)(slots[bad]))
        d = kk.KvAppendDesc()
        d.pools = kk.KvPools(p(micro), 0, 4, 0, 1, 1, D, 8)
        d.layer, d.rows, d.q_heads, d.rotary_dim = 0, 1, 1, D
        d.cos_sin, d.table_positions = p(cs), table
        d.slots, d.positions = p(one), p(pos) + 4 * bad
        d.query, d.key, d.value = p(x), p(x) + 2 * D, p(x) + 4 * D
        d.query_stride = d.key_stride = d.value_stride = 3 * D
        d.query_out, d.query_out_stride = p(out), D
        assert kk.kernels()["kv_append_rope"](C.byref(d), None) == 0
        torch.cuda.synchronize()
        assert kk.kernels()["device_status"](None) == codes[bad]
        if codes[bad]:
            assert bool((micro == 0).all()) and bool((out == 3.0).all())
        else:  # cos 1, sin 0: copied
            assert torch.equal(out[0], x[0, :D]) and int((micro != 0).sum()) == int((x[0, D:] != 0).sum())


@gpu_test
def test_append_behind_32_bit_offsets(kk):
    """Rows of queries, and a page, that begin more than 2^32 elements behind their arrays' start."""
    layers, page, hkv, hq, rows = 2, 64, 16, 2, 3
    slot, stride = 16400, (1 << 31) + 8
    pool = torch.empty(slot + 1, layers, 2, page, hkv, 64, dtype=torch.half, device="cuda")
    pool[slot:] = 7.0
    q = torch.empty(2 * stride + hq * 64, dtype=torch.half, device="cuda")
    rng = np.random.RandomState(20)
    x = rng.randn(rows, hq + 2 * hkv, 64).astype(np.float16)
    for r in range(rows):
        q[r * stride:r * stride + hq * 64] = torch.from_numpy(x[r, :hq].reshape(-1)).cuda()
    kv = torch.from_numpy(x[:, hq:].reshape(rows, -1)).cuda()
    slots = to_device_bytes((kk.KvSlot * rows)(*[kk.KvSlot(slot, t, 0, 1) for t in (63, 0, 5)]))
    positions = np.array([9, 1000, 3], np.uint32)
    d_pos = torch.from_numpy(positions.view(np.int32)).cuda()
    d = kk.KvAppendDesc()
    d.pools = kk.KvPools(p(pool), 0, slot + 1, 0, layers, hkv, 64, page)
    d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 1, rows, hq, 64, 10000.0
    d.slots, d.positions = p(slots), p(d_pos)
    d.query = d.query_out = p(q)
    d.query_stride = d.query_out_stride = stride
    d.key, d.value = p(kv), p(kv) + 2 * 64 * hkv
    d.key_stride = d.value_stride = kv.shape[1]
    torch.cuda.synchronize()
    assert kk.kernels()["kv_append_rope"](C.byref(d), None) == 0
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    got_q = np.stack([q[r * stride:r * stride + hq * 64].cpu().numpy() for r in range(rows)]).reshape(rows, hq, 64)
    page_now = pool[slot].cpu().numpy()
    got_k = page_now[1, 0, [63, 0, 5]]
    got = np.concatenate([got_q, got_k], 1)
    turned = x[:, :hq + hkv]
    ab = np.abs(turned[..., :32].astype(float)) + np.abs(turned[..., 32:].astype(float))
    assert_rounded(got, rotate_ref(turned, positions, 64, 10000.0), np.concatenate([ab, ab], -1))
    assert np.array_equal(page_now[1, 1, [63, 0, 5]], x[:, hq + hkv:])
    assert (page_now[0] == 7).all() and (np.delete(page_now[1], [63, 0, 5], 1) == 7).all()


@gpu_test
@pytest.mark.parametrize("theta", [1.0, 1.0001, 1.5, 5.0, 37.0, 10000.0, 1e6, 3e38])
@pytest.mark.parametrize("rotary", [64, 128, 256])
def test_append_angles_of_any_theta(kk, theta, rotary):
    """The farthest positions, where an error of a power of theta counts 2^32 times. The pairs are (1, 0) and
    (0, 1): the results are cosines and sines, and those near zero tell the angle to 4e-6 rad in FP16."""
    theta = float(np.float32(theta))
    rows, dim, half = 1024, 256, rotary // 2
    rng = np.random.RandomState(rotary)
    positions = rng.randint((1 << 32) - 100000, 1 << 32, rows, dtype=np.uint64).astype(np.uint32)
    positions[0] = 0xFFFFFFFF
    x = np.zeros((rows, 4, dim), np.float16)  # two query heads, a key and a value
    x[:, 0, :half] = x[:, 1, half:rotary] = x[:, 2, :half] = 1.0
    micro = torch.zeros(rows // 64, 1, 2, 64, 1, dim, dtype=torch.half, device="cuda")
    slots = to_device_bytes((kk.KvSlot * rows)(*[kk.KvSlot(r // 64, r % 64, 0, 1) for r in range(rows)]))
    d_x, d_pos = torch.from_numpy(x.reshape(rows, -1)).cuda(), torch.from_numpy(positions.view(np.int32)).cuda()
    out = torch.zeros(rows, 2 * dim, dtype=torch.half, device="cuda")
    d = kk.KvAppendDesc()
    d.pools = kk.KvPools(p(micro), 0, rows // 64, 0, 1, 1, dim, 64)
    d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 0, rows, 2, rotary, theta
    d.slots, d.positions = p(slots), p(d_pos)
    d.query, d.key, d.value = p(d_x), p(d_x) + 4 * dim, p(d_x) + 6 * dim
    d.query_stride = d.key_stride = d.value_stride = 4 * dim
    d.query_out, d.query_out_stride = p(out), 2 * dim
    torch.cuda.synchronize()
    assert kk.kernels()["kv_append_rope"](C.byref(d), None) == 0
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    got = np.concatenate([out.cpu().numpy().reshape(rows, 2, dim), micro[:, 0, 0].cpu().numpy().reshape(rows, 1, dim)], 1)
    size = np.zeros(got.shape)
    size[..., :rotary] = 1.0
    assert_rounded(got, rotate_ref(x[:, :3], positions, rotary, theta), size)


@gpu_test
def test_append_inputs_filled_again_as_a_programmatic_dependent(kk):
    """kk_fill_fp16 launched ahead of the append's end waits for it before it writes over the append's inputs."""
    rows, hq, hkv, D = 16384, 32, 8, 128
    width = (hq + 2 * hkv) * D
    K = kk.kernels()
    micro = torch.zeros(rows // 64, 1, 2, 64, hkv, D, dtype=torch.half, device="cuda")
    slots = to_device_bytes((kk.KvSlot * rows)(*[kk.KvSlot(r // 64, r % 64, 0, 1) for r in range(rows)]))
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    x, out = torch.empty(rows, width, dtype=torch.half, device="cuda"), torch.empty(rows, hq * D, dtype=torch.half, device="cuda")
    d = kk.KvAppendDesc()
    d.pools = kk.KvPools(p(micro), 0, rows // 64, 0, 1, hkv, D, 64)
    d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 0, rows, hq, D, 10000.0
    d.slots, d.positions = p(slots), p(pos)
    d.query, d.key, d.value = (p(x) + 2 * D * n for n in (0, hq, hq + hkv))
    d.query_stride = d.key_stride = d.value_stride = width
    d.query_out, d.query_out_stride = p(out), hq * D
    torch.cuda.synchronize()
    kept = []
    for pdl in (0, 1, 1, 1):
        assert K["fill_fp16"](p(x), x.numel(), 1, 1.0, None) == 0
        torch.cuda.synchronize()
        K["set_pdl"](pdl)
        assert K["kv_append_rope"](C.byref(d), None) == 0
        assert K["fill_fp16"](p(x), x.numel(), 2, 1.0, None) == 0
        K["set_pdl"](0)
        torch.cuda.synchronize()
        assert K["device_status"](None) == 0
        kept.append((out.clone(), micro.clone()))
    for a, b in kept[1:]:
        assert torch.equal(a, kept[0][0]) and torch.equal(b, kept[0][1])


@gpu_test
def test_append_calls_that_overlap_on_two_streams(kk):
    """Two batches into pages of their own, launched alternately on two streams with nothing in between."""
    K, D, built = kk.kernels(), 64, []
    for seed, (rows, hq, hkv) in enumerate(((3000, 8, 2), (700, 32, 4))):
        rng = np.random.RandomState(50 + seed)
        x = (rng.randn(rows, hq + 2 * hkv, D) * 2).astype(np.float16)
        positions = rng.randint(0, 1 << 20, rows).astype(np.uint32)
        arrays = [torch.from_numpy(x.reshape(rows, -1)).cuda(), torch.from_numpy(positions.view(np.int32)).cuda(),
                  to_device_bytes((kk.KvSlot * rows)(*[kk.KvSlot(r // 64, r % 64, 0, 1) for r in range(rows)])),
                  torch.zeros(rows, hq * D, dtype=torch.half, device="cuda"),
                  torch.zeros(rows // 64 + 1, 1, 2, 64, hkv, D, dtype=torch.half, device="cuda")]
        d = kk.KvAppendDesc()
        d.pools = kk.KvPools(p(arrays[4]), 0, rows // 64 + 1, 0, 1, hkv, D, 64)
        d.layer, d.rows, d.q_heads, d.rotary_dim, d.theta = 0, rows, hq, D, 10000.0
        d.slots, d.positions = p(arrays[2]), p(arrays[1])
        d.query, d.key, d.value = (p(arrays[0]) + 2 * D * n for n in (0, hq, hq + hkv))
        d.query_stride = d.key_stride = d.value_stride = (hq + 2 * hkv) * D
        d.query_out, d.query_out_stride = p(arrays[3]), hq * D
        built.append((x, positions, hq, hkv, arrays, d, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(20):
        for *_, d, stream in built:
            assert K["kv_append_rope"](C.byref(d), stream.cuda_stream) == 0
    torch.cuda.synchronize()
    assert K["device_status"](None) == 0
    for x, positions, hq, hkv, arrays, _, _ in built:
        rows = len(x)
        page = arrays[4][:, 0].cpu().numpy().transpose(1, 0, 2, 3, 4).reshape(2, -1, hkv, D)[:, :rows]
        got = np.concatenate([arrays[3].cpu().numpy().reshape(rows, hq, D), page[0]], 1)
        turned = x[:, :hq + hkv]
        ab = np.abs(turned[..., :32].astype(float)) + np.abs(turned[..., 32:].astype(float))
        assert_rounded(got, rotate_ref(turned, positions, D, 10000.0), np.concatenate([ab, ab], -1))
        assert np.array_equal(page[1], x[:, hq + hkv:])
