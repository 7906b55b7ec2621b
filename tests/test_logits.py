"""kk_logits_process: penalties, biases, grammar masks and the greedy token. The
refusals run on the CPU; the results run on the GPU and must equal the formula
evaluated in FP32 with one rounding per operation, bit for bit."""
import ctypes as C

import numpy as np
import pytest
import torch

from gpu_util import p

gpu = [pytest.mark.gpu, pytest.mark.skipif(not torch.cuda.is_available(), reason="needs a CUDA device")]
NONE = 0xFFFFFFFF


def gpu_test(fn):
    for mark in gpu:
        fn = mark(fn)
    return fn


def valid_desc(kk):
    d = kk.LogitsDesc()
    d.logits, d.out, d.tokens, d.logits_stride, d.out_stride = 1 << 20, 1 << 24, 1 << 16, 100, 100
    d.rows, d.vocab = 2, 100
    return d


@pytest.mark.parametrize("change", [
    dict(vocab=0), dict(logits=None), dict(out=None, tokens=None), dict(logits_stride=99), dict(out_stride=99),
    dict(out=1 << 20, out_stride=128), dict(logits=(1 << 20) + 2), dict(repetition=16), dict(presence=16),
    dict(frequency=16), dict(repetition=16, history_offsets=16, history_size=4),
    dict(bias_offsets=16, bias_size=3), dict(bias_offsets=16, bias_size=3, bias_tokens=16),
    dict(mask=16, mask_stride=3, num_masks=2), dict(vocab=(1 << 30) + 1, logits_stride=1 << 31, out_stride=1 << 31),
    dict(repetition=16, history_offsets=18, history=16, history_size=4), dict(repetition=17, history_offsets=16),
    dict(repetition=16, history_offsets=16, history=18, history_size=4), dict(bias_offsets=18),
    dict(bias_offsets=16, bias_tokens=18, bias_values=16, bias_size=1), dict(mask=18, mask_stride=4, num_masks=2),
    dict(mask=16, mask_stride=4, num_masks=2, mask_rows=17),
    dict(vocab=500000, logits_stride=500000, out_stride=500000, bias_offsets=16),
    dict(vocab=20000000, logits_stride=20000000, out_stride=20000000, mask=16, mask_stride=625000, num_masks=1),
], ids=str)
def test_logits_refuses(kk, change):
    d = valid_desc(kk)
    for name, value in change.items():
        setattr(d, name, value)
    assert kk.kernels()["logits_process"](C.byref(d), None) == kk.KK_EINVAL


@pytest.mark.parametrize("change", [
    dict(bias_offsets=16, bias_tokens=16, bias_values=16, bias_size=(1 << 32) - 255),
    dict(bias_offsets=16, bias_tokens=16, bias_values=16, bias_size=1 << 40),
    dict(repetition=16, history_offsets=16, history=16, history_size=(1 << 32) - 255),
    dict(repetition=16, history_offsets=16, history=16, history_size=1 << 33),
], ids=str)
def test_logits_refuses_lists_that_32_bit_indices_cannot_step_over(kk, change):
    """A row's list that ends within a step of 2^32 would be walked for ever."""
    d = valid_desc(kk)
    for name, value in change.items():
        setattr(d, name, value)
    assert kk.kernels()["logits_process"](C.byref(d), None) == kk.KK_EINVAL


def test_logits_without_rows_launches_nothing(kk):
    d = valid_desc(kk)
    d.rows = 0
    assert kk.kernels()["logits_process"](C.byref(d), None) == 0
    assert kk.kernels()["logits_process"](None, None) == kk.KK_EINVAL


class Case:
    """Host arrays of one call; `expect` evaluates the formula in FP32."""

    def __init__(self, rows, vocab, seed=0, stride=0, scale=3.0):
        self.rng = np.random.RandomState(seed)
        self.rows, self.vocab, self.stride = rows, vocab, stride or vocab
        self.logits = (self.rng.randn(rows, self.stride) * scale).astype(np.float32)
        self.history = self.prompts = self.factors = self.bias = self.mask = self.mask_rows = None

    def with_history(self, lens, prompts=None, repetition=True, presence=True, frequency=True):
        self.history = [self.rng.randint(0, max(1, self.vocab // (1 + i % 3)), n).astype(np.uint32)
                        for i, n in enumerate(lens)]
        self.prompts = None if prompts is None else np.asarray(prompts, np.uint32)
        u = lambda lo, hi: self.rng.uniform(lo, hi, self.rows).astype(np.float32)  # noqa: E731
        self.factors = [u(0.5, 2) if repetition else None, u(-1, 1) if presence else None, u(-0.5, 1) if frequency else None]
        return self

    def with_bias(self, counts):
        self.bias = []
        for n in counts:
            ids = np.sort(self.rng.choice(self.vocab, min(n, self.vocab), replace=False)).astype(np.uint32)
            self.bias.append((ids, (self.rng.randn(len(ids)) * 5).astype(np.float32)))
        return self

    def with_mask(self, density, masks=None, rows=None):
        n = masks or self.rows
        bits = self.rng.rand(n, -(-self.vocab // 32) * 32) < density
        self.mask = np.packbits(bits, axis=1, bitorder="little").view(np.uint32)
        self.mask_rows = None if rows is None else np.asarray(rows, np.uint32)
        return self

    def expect(self):
        x = self.logits[:, :self.vocab].copy()
        tokens = np.zeros(self.rows, np.int64)
        with np.errstate(all="ignore"):
            for r in range(self.rows):
                if self.history is not None:
                    rep, pres, freq = (np.float32(n) if f is None else f[r] for f, n in zip(self.factors, (1, 0, 0)))
                    text = self.history[r][self.history[r] < self.vocab]
                    given = self.history[r][0 if self.prompts is None else self.prompts[r]:]
                    seen = np.unique(text)
                    v = x[r, seen]
                    x[r, seen] = np.where(v > 0, v / rep, v * rep)
                    ids, n = np.unique(given[given < self.vocab], return_counts=True)
                    x[r, ids] = (x[r, ids] - (freq * n.astype(np.float32)).astype(np.float32)).astype(np.float32) - pres
                if self.bias is not None:
                    ids, values = self.bias[r]
                    last = {int(i): b for i, b in zip(ids, values) if i < self.vocab}
                    for i, b in last.items():
                        x[r, i] = x[r, i] + b
                if self.mask is not None:
                    m = r if self.mask_rows is None else int(self.mask_rows[r])
                    if m != NONE:
                        allowed = np.unpackbits(self.mask[m].view(np.uint8), bitorder="little")[:self.vocab]
                        x[r, allowed == 0] = -np.inf
                y = np.where(np.isnan(x[r]), -np.inf, x[r])
                tokens[r] = int(np.argmax(y)) if y.max() > -np.inf else NONE
        return x, tokens

    def call(self, kk, in_place=False, want_out=True, want_tokens=True, stream=None, offset=0):
        keep = []

        def up(a, dtype):
            t = torch.from_numpy(np.ascontiguousarray(a).view(dtype)).cuda()
            keep.append(t)
            return t

        def ragged(lists, dtype):
            offsets = np.concatenate([[0], np.cumsum([len(a) for a in lists])]).astype(np.uint32)
            flat = np.concatenate(lists) if lists and sum(map(len, lists)) else np.zeros(1, dtype)
            return up(flat, np.int32 if dtype == np.uint32 else np.float32), up(offsets, np.int32), int(offsets[-1])

        d = kk.LogitsDesc()
        room = torch.zeros(self.rows * self.stride + 8, device="cuda")
        x = room[offset:offset + self.rows * self.stride].view(self.rows, self.stride)
        x.copy_(torch.from_numpy(self.logits))
        out = x if in_place else torch.full_like(x, 9.0)
        tokens = torch.full((self.rows,), -7, dtype=torch.int32, device="cuda")
        d.logits, d.logits_stride, d.rows, d.vocab = p(x), self.stride, self.rows, self.vocab
        d.out, d.out_stride = p(out) if want_out else None, self.stride
        d.tokens = p(tokens) if want_tokens else None
        if self.history is not None:
            t, o, d.history_size = ragged(self.history, np.uint32)
            d.history, d.history_offsets = p(t), p(o)
            if self.prompts is not None:
                d.prompt_counts = p(up(self.prompts, np.int32))
            for name, f in zip(("repetition", "presence", "frequency"), self.factors):
                if f is not None:
                    setattr(d, name, p(up(f, np.float32)))
        if self.bias is not None:
            t, o, d.bias_size = ragged([b[0] for b in self.bias], np.uint32)
            v, _, _ = ragged([b[1] for b in self.bias], np.float32)
            d.bias_tokens, d.bias_values, d.bias_offsets = p(t), p(v), p(o)
        if self.mask is not None:
            d.mask, d.mask_stride, d.num_masks = p(up(self.mask, np.int32)), self.mask.shape[1], len(self.mask)
            if self.mask_rows is not None:
                d.mask_rows = p(up(self.mask_rows, np.int32))
        torch.cuda.synchronize()
        assert kk.kernels()["logits_process"](C.byref(d), stream.cuda_stream if stream else None) == 0
        torch.cuda.synchronize()
        return out.cpu().numpy(), tokens.cpu().numpy().view(np.uint32).astype(np.int64), keep

    def check(self, kk, in_place=False, want_out=True, want_tokens=True, status=0, **kw):
        out, tokens, _ = self.call(kk, in_place, want_out, want_tokens, **kw)
        assert kk.kernels()["device_status"](None) == status
        x, want = self.expect()
        if want_out:
            assert np.array_equal(out[:, :self.vocab], x, equal_nan=True)
            gap = self.logits[:, self.vocab:] if in_place else 9.0
            assert (out[:, self.vocab:] == gap).all()  # between the rows
        if want_tokens:
            assert np.array_equal(tokens, want), (tokens, want)
        else:
            assert (tokens == 0xFFFFFFF9).all()


SHAPES = [(1, 1), (3, 31), (2, 32), (5, 1000), (4, 4097), (1, 32000), (7, 50021), (2, 131072), (40, 9999), (1, 399999)]


@gpu_test
@pytest.mark.parametrize("rows,vocab", SHAPES)
@pytest.mark.parametrize("parts", ["none", "history", "bias", "mask", "all"])
def test_logits_equal_formula(kk, rows, vocab, parts):
    c = Case(rows, vocab, seed=rows + vocab)
    if parts in ("history", "all"):
        lens = c.rng.randint(0, 5000, rows)
        lens[0] = 3 if rows > 1 else 4999
        c.with_history(lens, prompts=(lens * c.rng.rand(rows)).astype(int))
    if parts in ("bias", "all"):
        c.with_bias(c.rng.randint(0, 400, rows))
    if parts in ("mask", "all"):
        c.with_mask(0.5)
    if parts == "all" and vocab > 300000:
        c.with_history([2000], prompts=[0])
    c.check(kk)


@gpu_test
@pytest.mark.parametrize("kw", [dict(in_place=True), dict(want_out=False), dict(want_tokens=False), dict(offset=1),
                                dict(offset=3, in_place=True)], ids=str)
@pytest.mark.parametrize("vocab,stride", [(5003, 5003), (5003, 5120), (33001, 33002)])
def test_logits_forms(kk, kw, vocab, stride):
    c = Case(6, vocab, seed=1, stride=stride)
    c.with_history([0, 1, 17, 300, 4000, 9000], prompts=[0, 1, 3, 300, 0, 8000]).with_bias([0, 1, 3, 50, 500, 5003])
    c.with_mask(0.7, masks=3, rows=[0, NONE, 2, 1, 1, NONE])
    c.check(kk, **kw)


@gpu_test
@pytest.mark.parametrize("which", range(3))
def test_logits_single_factors_and_no_prompt_counts(kk, which):
    c = Case(4, 6001, seed=which)
    c.with_history([100, 0, 2000, 1], None, *[i == which for i in range(3)])
    c.check(kk)


@gpu_test
def test_logits_specials_masks_and_ties(kk):
    vocab = 9000
    c = Case(9, vocab, seed=4)
    x = c.logits
    x[0] = -np.inf                                   # nothing to choose
    x[1] = np.nan                                    # nothing to choose
    x[2, [77, 5000, 8999]] = 1e30                    # ties: the lowest id
    x[3] = 0.0
    x[3, 0] = -0.0                                   # -0 equals +0: id 0
    x[4, 123] = np.nan                               # masked below
    x[4, 124] = np.inf                               # masked below
    x[5, 4000] = np.inf
    x[6] = np.finfo(np.float32).min                  # the type's lowest value can be chosen
    x[7, 17] = np.nan
    c.with_mask(2.0)
    c.mask[8] = 0                                    # a mask that leaves nothing
    c.mask[4, 123 // 32] &= ~np.uint32(1 << (123 % 32))
    c.mask[4, 124 // 32] &= ~np.uint32(1 << (124 % 32))
    c.check(kk)
    _, tokens = c.expect()
    assert list(tokens[[0, 1, 2, 3, 6, 8]]) == [NONE, NONE, 77, 0, 0, NONE]
    c.with_history([50] * 9, prompts=[25] * 9).with_bias([60] * 9)
    c.check(kk)


@gpu_test
@pytest.mark.parametrize("rows,vocab,lens", [
    (2, 33000, (70001, 65536)),      # counts beyond 16 bits
    (3, 50021, (30000, 65535, 90000)),  # more distinct tokens than a list of them holds
    (2, 300, (66000, 1)), (1, 4097, (131072,)), (2, 131072, (131072, 20)),
], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_logits_long_histories(kk, rows, vocab, lens, in_place):
    c = Case(rows, vocab, seed=vocab, stride=vocab + 1)
    c.with_history(lens, prompts=[min(n // 50, 100) for n in lens]).with_mask(0.8)
    c.history[0][:66000] = vocab // 3  # one token, more often than 16 bits count
    c.with_bias([vocab // 2, 0, 40][:rows])
    c.check(kk, in_place=in_place)


@gpu_test
def test_logits_repeated_ids_and_ids_outside_the_vocabulary(kk):
    c = Case(3, 5000, seed=6)
    c.with_history([4000, 4000, 4000], prompts=[0, 4000, 2000])
    for h in c.history:
        h[::2] = 4321                                # one token, 2000 times
        h[1::7] = 5000                               # outside
        h[2::9] = NONE
    c.bias = [(np.array([5, 5, 5, 4321, 4321, 6000], np.uint32), np.arange(6, dtype=np.float32))] * 3
    c.check(kk)


@gpu_test
def test_logits_reports_bad_lists(kk):
    bad = 3
    c = Case(2, 700, seed=7).with_history([10, 10])
    c.history = [np.zeros(0, np.uint32)] * 2          # expected: left out
    _, want = c.expect()
    d_offsets = torch.tensor([5, 3, 99], dtype=torch.int32).cuda()  # decreases; passes the array
    for which in ("history", "bias"):
        d = kk.LogitsDesc()
        x = torch.from_numpy(c.logits).cuda()
        tokens = torch.zeros(2, dtype=torch.int32, device="cuda")
        ids = torch.zeros(10, dtype=torch.int32, device="cuda")
        values = torch.ones(10, device="cuda")
        d.logits = d.out = p(x)
        d.logits_stride = d.out_stride = d.vocab = 700
        d.rows, d.tokens = 2, p(tokens)
        if which == "history":
            d.history, d.history_offsets, d.history_size, d.presence = p(ids), p(d_offsets), 10, p(values)
        else:
            d.bias_tokens, d.bias_values, d.bias_offsets, d.bias_size = p(ids), p(values), p(d_offsets), 10
        assert kk.kernels()["logits_process"](C.byref(d), None) == 0
        torch.cuda.synchronize()
        assert kk.kernels()["device_status"](None) == bad
        assert torch.equal(x, torch.from_numpy(c.logits).cuda()) and list(tokens.cpu().numpy()) == list(want)
    c = Case(2, 700, seed=8).with_mask(1.0, masks=2, rows=[2, 1])
    out, tokens, _ = c.call(kk)
    assert kk.kernels()["device_status"](None) == bad
    assert np.isneginf(out[0]).all() and tokens[0] == NONE and np.array_equal(out[1], c.logits[1])
    c = Case(1, 700, seed=9)
    c.bias = [(np.array([9, 3], np.uint32), np.ones(2, np.float32))]  # descends
    c.call(kk)
    assert kk.kernels()["device_status"](None) == bad


@gpu_test
def test_logits_on_streams_captured_and_repeated(kk):
    """Two streams at once, and one captured call replayed on new logits."""
    cases = [Case(20, 20011, seed=s).with_history([900] * 20, prompts=[100] * 20).with_bias([9] * 20).with_mask(0.9)
             for s in (1, 2)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for c, s in zip(cases, streams):
        c.check(kk, stream=s)
    x = torch.zeros(3, 40000, device="cuda")
    out, tokens = torch.empty_like(x), torch.zeros(3, dtype=torch.int32, device="cuda")
    d = kk.LogitsDesc()
    d.logits, d.out, d.tokens, d.rows, d.vocab = p(x), p(out), p(tokens), 3, 40000
    d.logits_stride = d.out_stride = 40000
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert kk.kernels()["logits_process"](C.byref(d), torch.cuda.current_stream().cuda_stream) == 0
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, x) and torch.equal(tokens.long(), x.argmax(-1))


@gpu_test
def test_logits_behind_32_bit_offsets(kk):
    """Rows that begin more than 2^32 elements behind the array's start (17 GB), in place."""
    rows, vocab, stride = 3, 5000, (1 << 31) + 1
    x = torch.empty(2 * stride + vocab, device="cuda")
    rng = np.random.RandomState(21)
    host = rng.randn(rows, vocab).astype(np.float32)
    for r in range(rows):
        x[r * stride:r * stride + vocab] = torch.from_numpy(host[r]).cuda()
    banned = torch.tensor([int(t) for t in host.argmax(1)], dtype=torch.int32, device="cuda")
    offsets = torch.arange(rows + 1, dtype=torch.int32, device="cuda")
    values = torch.full((rows,), -100.0, device="cuda")
    tokens = torch.zeros(rows, dtype=torch.int32, device="cuda")
    d = kk.LogitsDesc()
    d.logits = d.out = p(x)
    d.logits_stride = d.out_stride = stride
    d.rows, d.vocab, d.tokens = rows, vocab, p(tokens)
    d.bias_tokens, d.bias_values, d.bias_offsets, d.bias_size = p(banned), p(values), p(offsets), rows
    torch.cuda.synchronize()
    assert kk.kernels()["logits_process"](C.byref(d), None) == 0
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    for r in range(rows):
        host[r, host[r].argmax()] += np.float32(-100.0)
        assert np.array_equal(x[r * stride:r * stride + vocab].cpu().numpy(), host[r])
    assert np.array_equal(tokens.cpu().numpy(), host.argmax(1))


@gpu_test
@pytest.mark.parametrize("history", [0, 70000], ids=["alone", "with_history"])
@pytest.mark.parametrize("ids", ["shuffled", "one_id_and_others"])
def test_logits_descending_bias_ids_stay_in_their_row(kk, history, ids):
    """Biases out of order, ids again and again: reported, and whatever the row gets of them, tokens without a
    bias and the other rows are as they would be."""
    vocab = 20000
    c = Case(3, vocab, seed=30)
    if history:
        c.with_history([50, history, 0], prompts=[0, 100, 0])
    c.with_bias([300, 0, 70])
    n = 6000
    named = c.rng.randint(0, 3000, n).astype(np.uint32)
    if ids == "one_id_and_others":
        named[::2] = 1234
    c.bias[1] = (named, np.ones(n, np.float32))
    for _ in range(3):
        out, tokens, _ = c.call(kk)
        assert kk.kernels()["device_status"](None) == 3
        x, want = c.expect()
        free = np.setdiff1d(np.arange(vocab), named)
        assert np.array_equal(out[[0, 2]], x[[0, 2]]) and np.array_equal(tokens[[0, 2]], want[[0, 2]])
        assert np.array_equal(out[1, free], x[1, free])
        assert np.isfinite(out[1]).all()
        assert tokens[1] == int(np.argmax(out[1]))


@gpu_test
@pytest.mark.parametrize("vocab,masked", [(400000, False), (400001, True), (400003, False), (9999999, True), (10000000, True),
                                          (10000001, False), (40000003, False)], ids=str)
@pytest.mark.parametrize("in_place", [False, True])
def test_logits_vocabularies_beyond_the_listed_tokens(kk, vocab, masked, in_place):
    """Without history and biases nothing is counted: the vocabulary may be larger, up to 10 million with a mask."""
    c = Case(2 if vocab < 10 ** 6 else 1, vocab, seed=vocab % 1000, stride=vocab + 3)
    c.logits[0, [vocab - 1, vocab // 2]] = 100.0
    if masked:
        c.with_mask(0.5)
        c.mask[0, vocab // 2 // 32] &= ~np.uint32(1 << (vocab // 2 % 32))
        c.mask[0, (vocab - 1) // 32] |= np.uint32(1 << ((vocab - 1) % 32))
    c.check(kk, in_place=in_place, offset=1)
    assert c.expect()[1][0] == (vocab - 1 if masked else vocab // 2)


@pytest.mark.parametrize("vocab,kw", [
    (400001, dict(bias_offsets=16)), (400001, dict(repetition=16, history_offsets=16)),
    (10000001, dict(mask=16, mask_stride=1 << 20, num_masks=1)), ((1 << 30) + 1, {}),
], ids=str)
def test_logits_refuses_vocabularies_beyond_their_limits(kk, vocab, kw):
    d = valid_desc(kk)
    d.vocab, d.logits_stride, d.out_stride = vocab, 1 << 31, 1 << 31
    for name, value in kw.items():
        setattr(d, name, value)
    assert kk.kernels()["logits_process"](C.byref(d), None) == kk.KK_EINVAL


@gpu_test
def test_logits_calls_that_overlap_on_two_streams(kk):
    """Everything is built first; then calls are launched alternately on two streams, with nothing in between."""
    built = []
    for seed, (rows, vocab, history) in enumerate(((20, 20011, 900), (64, 32000, 4000))):
        c = Case(rows, vocab, seed=40 + seed).with_history([history] * rows, prompts=[100] * rows).with_bias([9] * rows)
        c.with_mask(0.9)
        up = lambda a, t: torch.from_numpy(np.ascontiguousarray(a).view(t)).cuda()  # noqa: E731
        ends = lambda lists: np.cumsum([0] + [len(a) for a in lists]).astype(np.uint32)  # noqa: E731
        arrays = dict(logits=up(c.logits, np.float32), history=up(np.concatenate(c.history), np.int32),
                      history_offsets=up(ends(c.history), np.int32), prompt_counts=up(c.prompts, np.int32),
                      repetition=up(c.factors[0], np.float32), presence=up(c.factors[1], np.float32),
                      frequency=up(c.factors[2], np.float32), bias_tokens=up(np.concatenate([b[0] for b in c.bias]), np.int32),
                      bias_values=up(np.concatenate([b[1] for b in c.bias]), np.float32),
                      bias_offsets=up(ends([b[0] for b in c.bias]), np.int32), mask=up(c.mask, np.int32),
                      out=torch.zeros(rows, vocab, device="cuda"), tokens=torch.zeros(rows, dtype=torch.int32, device="cuda"))
        d = kk.LogitsDesc()
        for name, t in arrays.items():
            setattr(d, name, p(t))
        d.logits_stride = d.out_stride = d.vocab = vocab
        d.rows, d.history_size, d.bias_size = rows, len(arrays["history"]), len(arrays["bias_tokens"])
        d.mask_stride, d.num_masks = c.mask.shape[1], rows
        built.append((c, d, arrays, torch.cuda.Stream()))
    torch.cuda.synchronize()
    call = kk.kernels()["logits_process"]
    for _ in range(20):
        for c, d, arrays, stream in built:
            assert call(C.byref(d), stream.cuda_stream) == 0
    torch.cuda.synchronize()
    assert kk.kernels()["device_status"](None) == 0
    for c, d, arrays, _ in built:
        x, want = c.expect()
        assert np.array_equal(arrays["out"].cpu().numpy(), x)
        assert np.array_equal(arrays["tokens"].cpu().numpy(), want)
