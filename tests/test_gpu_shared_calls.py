"""Calls of the shared-prompt operators that follow one another on one handle, and
arguments at the ends of their ranges, against plain models.

Bars.  Ids, adjusted logits and products are exact by definition.  A
log-probability is a float64 sum whose terms e^x are each off by at most 4e-11
of themselves; a term is scaled by such a factor again when its thread, wave,
workgroup and row find larger maxima, at most once a segment of 4096 ids of its
workgroup and three times in the joins, and the float64 sum over v terms rounds
within v 2^-53: (4 + segments) 4e-11 + v 2^-53, which for the vocabularies here
(25 segments, of which a workgroup takes at most two: 2.4e-10 and 1.1e-11) stays
below 2.6e-10, relative to 1 + |log-probability| for its last subtractions.
"""

import ctypes as C
import sys

import numpy as np
import pytest
import torch

from helpers import DeviceArray
from needle_hip import (HipKvCache, HipRows, HipSelector, HipSharedAttention, Int8Matrix,
                        NeedleError)
from needle_hip import lib as L
from needle_hip.models import DecoderGeometry, DecoderWeights, HipBatch, HipDecoder
from test_gpu_shared import adjusted_oracle, check_choice, choice_oracle, quantized

pytestmark = pytest.mark.gpu
LP_BAR = 2.6e-10


def say(*args):
    print("[case]", *args, file=sys.stderr, flush=True)


class Choice:
    """One adjusted selection on device arrays, its results filled with values that no
    selection gives before every call."""

    def __init__(self, rng, rows, v):
        self.rows, self.v = rows, v
        self.logits = (rng.standard_normal((rows, v)) * 4).astype(np.float32)
        self.told = dict(history=rng.integers(0, v, (rows, 90)).astype(np.uint32),
                         repetition=rng.uniform(1.0, 1.5, rows).astype(np.float32),
                         frequency=rng.uniform(0.0, 0.5, rows).astype(np.float32))
        self.dl = DeviceArray(self.logits)
        self.arrays = {k: DeviceArray(a) for k, a in self.told.items()}
        self.adjust = L.LogitAdjust()
        for name, a in self.arrays.items():
            setattr(self.adjust, name, a.ptr.value)
        self.adjust.history_stride = 90
        self.want = [choice_oracle(adjusted_oracle(self.logits, r, self.told), np.ones(v, bool))
                     for r in range(rows)]

    def run(self, hip, selector):
        ids = DeviceArray(np.full(self.rows, 0x5A5A5A5A, np.uint32))
        lps = DeviceArray(np.full(self.rows, 1e300))
        selector.run(self.dl.ptr.value, self.rows, self.v, ids.ptr.value, lps.ptr.value, self.adjust)
        hip._check(hip.lib.nd_sync(hip.ctx))
        got = ids.read(), lps.read()
        ids.free(), lps.free()
        return got

    def check(self, got):
        for r, (pick, lp) in enumerate(self.want):
            assert got[0][r] == pick, (r, got[0][r], pick)
            assert abs(got[1][r] - lp) <= LP_BAR * (1 + abs(lp)), (r, got[1][r], lp)

    def free(self):
        for a in [self.dl, *self.arrays.values()]:
            a.free()


@pytest.mark.parametrize("xcd_local", [True, False])
def test_one_selector_for_batches_of_changing_size(hip, rng, xcd_local):
    """A batch that shrinks as its answers end, and grows again: every row of every call is
    chosen, with the bits of a selector of its own."""
    say("selector sizes", xcd_local)
    calls = [Choice(rng, rows, v) for rows, v in
             ((9, 8192), (4, 8192), (1, 8192), (8, 30000), (9, 30000), (2, 100000), (3, 4097),
              (64, 32768), (40, 32768), (1, 32768), (5, 100))]
    probed = C.c_uint32()
    selector = HipSelector(hip, 70)
    try:
        hip._check(hip.lib.nd_test_xcd_local(hip.ctx, int(xcd_local), C.byref(probed)))
        for turn in (calls, calls[::-1], calls):
            for call in turn:
                got = call.run(hip, selector)
                call.check(got)
                own = HipSelector(hip, call.rows)
                alone = call.run(hip, own)
                own.free()
                assert np.array_equal(got[0], alone[0]) and np.array_equal(got[1], alone[1])
    finally:
        hip._check(hip.lib.nd_test_xcd_local(hip.ctx, 1, C.byref(probed)))
    selector.free()
    for call in calls:
        call.free()


def test_infinite_penalties_reach_generated_tokens_only(hip, rng):
    """An infinite frequency or presence penalty bars what was generated and leaves ids of
    the prompt, of the biases and of no list as they are."""
    say("infinite penalties")
    v, n, prompt = 9000, 60, 30
    logits = (rng.standard_normal((6, v)) * 4).astype(np.float32)
    history = rng.integers(0, v, (6, n)).astype(np.uint32)
    history[:, 0] = 0  # the first id is of the prompt
    history[:, 40] = logits.argmax(1)  # the best one was generated
    a = dict(history=history, prompt_lengths=np.full(6, prompt, np.uint32),
             frequency=np.array([np.inf, np.inf, 0.3, -np.inf, np.inf, 0], np.float32),
             presence=np.array([0.1, np.inf, np.inf, 0, 0, -np.inf], np.float32),
             bias_ids=rng.integers(0, v, (6, 9)).astype(np.uint32),
             bias=rng.standard_normal((6, 9)).astype(np.float32))
    ok = rng.random((6, v)) < 0.3
    ok[4:, 0] = True
    with np.errstate(all="ignore"):
        check_choice(hip, logits, a, None)
        check_choice(hip, logits, a, ok)


def test_batch_knows_its_prefix_cache_from_a_later_one_at_its_address(hip):
    say("prefix cache replaced")
    g = DecoderGeometry(layers=2, vocab=512)
    dec = HipDecoder(hip, DecoderWeights(g, 3))
    batch = HipBatch(dec, 2, 16)
    first = HipKvCache(hip, 2, 8, 32)
    batch.set_prefix(first, 32)
    batch.set_state([1, 2], [0, 0])
    batch.step(0)
    hip._check(hip.lib.nd_sync(hip.ctx))
    address = first.handle.value
    first.free()
    later = []
    while len(later) < 64 and address not in [c.handle.value for c in later]:
        later.append(HipKvCache(hip, 2, 8, 32))
    with pytest.raises(NeedleError) as e:
        batch.step(1)
    assert e.value.code == "INVALID_CACT"
    batch.set_prefix(later[-1], 32)
    batch.step(1)
    hip._check(hip.lib.nd_sync(hip.ctx))
    for x in [batch, dec] + later:
        x.free()


# Every form of the product's kernels: few rows, split tiles, whole tiles, k of two blocks.
@pytest.mark.parametrize("m,n,k", [(1, 301, 4096), (7, 16386, 128), (33, 64, 512), (65, 129, 128),
                                   (300, 516, 2048), (128, 2048, 256), (64, 16500, 128), (180, 33001, 512),
                                   (2050, 3088, 512), (2050, 3085, 512), (1025, 1600, 128)])
def test_products_take_the_roundings_they_are_defined_by(hip, rng, m, n, k):
    """y = add + ((float)sum s_n) s_m, each step rounded to float32: the same bits from
    every form."""
    say("product roundings", m, n, k)
    w = rng.integers(-128, 128, (n, k)).astype(np.int8)
    sw = rng.uniform(0.001, 0.02, n).astype(np.float32)
    x = (rng.standard_normal((m, k)) * rng.uniform(0.01, 10, (m, 1))).astype(np.float32)
    add = rng.standard_normal((m, n)).astype(np.float32)
    codes, scales = quantized(x)
    total = codes.astype(np.float32) @ w.T.astype(np.float32) if k * 2 ** 14 <= 2 ** 24 else (
        codes.astype(np.float64) @ w.T.astype(np.float64))  # exact either way
    want = total.astype(np.float32) * sw[None, :] * scales[:, None]
    mat = hip.upload(Int8Matrix(w, sw.reshape(n, 1), k))
    rows, dx = HipRows(hip, m, k), DeviceArray(x)
    rows.quantize(dx.ptr.value, m)
    y, a = DeviceArray(np.full((m, n), np.nan, np.float32)), DeviceArray(add)
    rows.matmul(mat, y.ptr.value)
    rows.matmul(mat, a.ptr.value, add=a.ptr.value)
    hip._check(hip.lib.nd_sync(hip.ctx))
    assert np.array_equal(y.read(), want)
    assert np.array_equal(a.read(), add + want)
    for d in (dx, y, a, rows):
        d.free()


@pytest.mark.parametrize("v", [1, 2, 3, 5, 31, 32, 33])
def test_selections_over_the_smallest_vocabularies(hip, rng, v):
    say("small vocabulary", v)
    logits = rng.standard_normal((3, v)).astype(np.float32)
    a = dict(history=rng.integers(0, v + 1, (3, 7)).astype(np.uint32),
             repetition=np.full(3, 1.5, np.float32), presence=np.full(3, 0.25, np.float32))
    check_choice(hip, logits, a, None)
    check_choice(hip, logits, a, np.eye(3, v, dtype=bool))


def test_captured_selections_share_a_selector(hip, rng):
    """Two captured selections of different batches on one selector, replayed in turn with
    eager ones of a third between them, on one stream: each gives what it gives alone."""
    say("captured selections")
    calls = [Choice(rng, rows, v) for rows, v in ((9, 30000), (4, 8192), (6, 20000))]
    selector = HipSelector(hip, 12)
    stream = torch.cuda.Stream()
    outs, graphs = [], []
    for call in calls:
        outs.append((torch.zeros(call.rows, dtype=torch.int32, device="cuda"),
                     torch.zeros(call.rows, dtype=torch.float64, device="cuda")))

    def enqueue(i):
        call, (ids, lps) = calls[i], outs[i]
        selector.run(call.dl.ptr.value, call.rows, call.v, ids.data_ptr(), lps.data_ptr(), call.adjust,
                     stream=stream.cuda_stream)

    torch.cuda.synchronize()
    for i in range(3):
        enqueue(i)
    stream.synchronize()
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            enqueue(i)
        graphs.append(graph)
    for turn in range(4):
        for i in (0, 2, 1, 0, 1, 2):
            for t in outs[i]:
                t.fill_(-7)
            torch.cuda.synchronize()
            if i < 2:
                with torch.cuda.stream(stream):
                    graphs[i].replay()
            else:
                enqueue(i)
            stream.synchronize()
            calls[i].check([t.cpu().numpy() for t in outs[i]])
    selector.free()
    for call in calls:
        call.free()


def test_rows_and_attention_workspaces_take_calls_of_changing_size(hip, rng):
    """One handle of rows for 40, 1, 17 and 40 rows, one attention workspace for long and
    short ranges in turn: the bits of handles of their own."""
    say("workspaces of changing size")
    k, n = 256, 515
    w = rng.integers(-127, 128, (n, k)).astype(np.int8)
    mat = hip.upload(Int8Matrix(w, np.full((n, 1), 0.01, np.float32), k))
    x = rng.standard_normal((40, k)).astype(np.float32)
    x[30] = np.inf  # what the larger call leaves behind the smaller one's rows
    d, y = DeviceArray(x), DeviceArray(np.zeros((40, n), np.float32))
    rows = HipRows(hip, 40, k)

    def product(handle, m):
        handle.quantize(d.ptr.value, m)
        handle.matmul(mat, y.ptr.value)
        hip._check(hip.lib.nd_sync(hip.ctx))
        return y.read()[:m]

    for m in (40, 1, 17, 40, 33):
        got = product(rows, m)
        own = HipRows(hip, m, k)
        assert np.array_equal(got, product(own, m), equal_nan=True), m
        own.free()
    batch, heads = 20, 2
    p, o = HipKvCache(hip, 1, heads, 3000), HipKvCache(hip, 1, batch * heads, 500)
    p.store(0, 0, *rng.standard_normal((2, 3000, heads, 64)).astype(np.float32))
    o.store(0, 0, *rng.standard_normal((2, 500, batch * heads, 64)).astype(np.float32))
    q = rng.standard_normal((batch, 2 * heads, 64)).astype(np.float32)
    shared = HipSharedAttention(hip, batch, heads, 2 * heads)
    for prefix, longest in ((3000, 500), (10, 1), (0, 0), (3000, 0), (0, 500), (64, 33), (3000, 500)):
        lengths = np.minimum(longest, rng.integers(0, longest + 1, batch))
        own = HipSharedAttention(hip, batch, heads, 2 * heads)
        assert np.array_equal(shared.attention(p, prefix, o, lengths, 0, q),
                              own.attention(p, prefix, o, lengths, 0, q)), (prefix, longest)
        own.free()
    for h in (rows, d, y, shared, p, o):
        h.free()
