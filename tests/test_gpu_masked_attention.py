"""Attention under masks (zdraw_hip_run_attention_masked) against the definition in 64 bits.

Tolerances count roundings (tests/rangeref.py, tolerance): half a step of the 16-bit output, half a step on every
probability, f32 in between."""
import ctypes as C

import numpy as np
import pytest

from tests import rangeref as rr
from zdraw_amd import hip, host

pytestmark = pytest.mark.gpu
D = 128
POISON = 0x7E55  # a NaN in either type


@pytest.fixture(scope="module")
def ctx():
    c = host.Context.init()
    yield c
    c.deinit()


class Call:
    """One call's operands. docs: lengths of the packed documents, per segment; key_docs: of their keys."""

    def __init__(self, ctx, q=1, k=None, *, batch=1, heads=4, kv=2, causal=True, docs=None, key_docs=None, prefix=None, cap=0.0, slopes=False,
                 scale=0.0, dtype=hip.BF16, pad=(0, 0, 0), off=0, seed=0, loud=1.0, x=None):
        k = q if k is None else k
        self.ctx, self.dtype, self.causal, self.cap, self.scale = ctx, dtype, causal, cap, scale
        self.shape, self.kshape = (batch, q, heads, D), (batch, k, kv, D)
        rng = np.random.default_rng(seed + 7 * q + k + heads)
        draw = lambda s, c: rr.bits(rng.standard_normal(s, dtype=np.float32) * c, dtype)
        self.q, self.k, self.v = draw(self.shape, 1.2 * loud), draw(self.kshape, 1.0), draw(self.kshape, 1.0)
        if x:
            x(self)
        self.slopes = np.float32(2.0) ** -np.arange(1, heads + 1, dtype=np.float32) if slopes else None
        self.starts = None if docs is None else np.array([np.concatenate(([0], np.cumsum(d))) for d in docs], np.uint32)
        self.kstarts = self.starts if key_docs is None else np.array([np.concatenate(([0], np.cumsum(d))) for d in key_docs], np.uint32)
        self.prefix = None if prefix is None else np.array(prefix, np.uint32).reshape(batch, -1)
        p, o = hip.MaskedAttn(), hip.MaskOperands()
        p.batch, p.q_tokens, p.k_tokens, p.heads, p.kv_heads, p.head_dim, p.dtype = batch, q, k, heads, kv, D, dtype
        p.causal, p.scale, p.softcap = int(causal), scale, cap
        p.documents = 0 if docs is None else len(docs[0])
        self.p, self.o, self.keep = p, o, []
        self.bufs = []
        for name, data, dst in (("q", self.q, p.q_stride), ("k", self.k, p.k_stride), ("v", self.v, p.v_stride)):
            size = rr.dense(dst, data.shape, pad)
            flat = np.concatenate((np.full(off, POISON, np.uint16), rr.spread(data, dst, size, np.uint16(POISON)), np.full(8, POISON, np.uint16)))
            setattr(p, name + "_off", 2 * off)
            self.bufs.append(ctx.buffer(flat))
        self.size = rr.dense(p.out_stride, self.shape, pad)
        p.out_off = 2 * off
        self.off = off
        self.out = ctx.buffer(np.full(off + self.size + 8, POISON, np.uint16))
        for name, a in (("q_starts", self.starts), ("prefix", self.prefix), ("slopes", self.slopes)):
            if a is not None:
                self.keep.append(ctx.buffer(a))
                setattr(o, name, self.keep[-1].handle)
        if key_docs is not None:
            self.keep.append(ctx.buffer(self.kstarts))
            o.k_starts = self.keep[-1].handle

    def args(self):
        return (*(b.handle for b in self.bufs), self.out.handle, C.byref(self.p), C.byref(self.o))

    def rc(self, queue=None):
        return hip.lib().zdraw_hip_run_attention_masked(queue or self.ctx.queue, *self.args())

    def enqueue(self, batch):
        return hip.lib().zdraw_hip_run_attention_masked_enc(batch, *self.args())

    def clear(self):
        self.out.write(np.full(self.off + self.size + 8, POISON, np.uint16))

    def read(self):
        """The output's bits; what lies between its rows has to be as it was."""
        flat = self.out.read(np.uint16, self.off + self.size + 8)
        got = rr.gather(flat[self.off:], self.p.out_stride, self.shape)
        rest = flat.copy()
        mask = rr.spread(np.ones(self.shape, np.uint16), self.p.out_stride, self.size, np.uint16(0))
        assert (rest[self.off:self.off + self.size][mask == 0] == POISON).all() and (rest[:self.off] == POISON).all()
        assert (rest[self.off + self.size:] == POISON).all()
        return got

    def want(self):
        batch, n, heads, _ = self.shape
        keys = self.kshape[1]
        out, absolute = np.zeros(self.shape), np.zeros(self.shape)
        live = np.zeros((batch, n), bool)
        f = lambda b: rr.value(b, self.dtype)
        for b in range(batch):
            starts, kstarts = (self.starts[b], self.kstarts[b]) if self.starts is not None else ([0, n], [0, keys])
            for d in range(len(starts) - 1):
                q0, q1, k0, k1 = int(starts[d]), int(starts[d + 1]), int(kstarts[d]), int(kstarts[d + 1])
                nk = k1 - k0
                pos = np.arange(q1 - q0) + nk - (q1 - q0)
                j = np.arange(nk)
                pre = int(self.prefix[b, d]) if self.prefix is not None else 0
                seen = np.ones((q1 - q0, nk), bool) if not self.causal else (j[None] <= pos[:, None]) | (j[None] < pre)
                out[b, q0:q1], absolute[b, q0:q1] = rr.rows(f(self.q[b, q0:q1]), f(self.k[b, k0:k1]), f(self.v[b, k0:k1]), seen, pos, self.scale, self.cap,
                                                            self.slopes)
                live[b, q0:q1] = True
        return out, absolute, live

    def check(self, what="", scores=32.0, run=True):
        if run:
            rc = self.rc()
            assert rc == 0, hip.last_error()
        got = self.read()
        want, absolute, live = self.want()
        assert (got[~live] == POISON).all(), f"{what}: rows outside of every document were written"
        rr.check(rr.value(got, self.dtype)[live], want[live], absolute[live], self.dtype, what, scores)
        return got


def say(*a):
    print(*a, flush=True)


# one row, the borders of a wave's 32 rows, of a block's 32 keys and of a workgroup's 128 rows; groups of one to five heads
@pytest.mark.parametrize("dtype", [hip.BF16, hip.F16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("q,heads,kv", [(1, 4, 2), (2, 1, 1), (31, 2, 2), (32, 2, 1), (33, 3, 1), (64, 5, 1), (77, 4, 2), (129, 3, 3), (257, 2, 2)])
def test_self_attention(ctx, q, heads, kv, causal, dtype):
    say(q, heads, kv, causal, dtype)
    Call(ctx, q, heads=heads, kv=kv, causal=causal, dtype=dtype).check()


# few queries at the end of many keys, keys fewer than queries (the first rows see none), no keys at all
@pytest.mark.parametrize("q,k,heads,kv", [(1, 2, 4, 2), (1, 1000, 8, 1), (3, 777, 4, 4), (40, 33, 2, 1), (200, 1, 2, 2), (5, 0, 2, 1), (300, 512, 2, 2), (2, 5000, 16, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_of_another_length(ctx, q, k, heads, kv, causal):
    say(q, k, heads, kv, causal)
    c = Call(ctx, q, k, heads=heads, kv=kv, causal=causal)
    got = c.check()
    if causal and k < q:
        assert (got[:, :q - k] == 0).all()


# many rows, so that the waves share key blocks (128 rows a workgroup): more than 1024 tiles of 32 rows
MANY = dict(heads=56, kv=56)  # of 650 rows: 1176 tiles


@pytest.mark.parametrize("dtype", [hip.BF16, hip.F16])
@pytest.mark.parametrize("causal,docs,prefix,cap,slopes", [(True, None, None, 0.0, False), (False, None, None, 0.0, False), (True, None, [[400]], 0.0, False),
                                                           (True, None, None, 20.0, True), (False, None, None, 0.0, True), (True, None, [[300]], 0.0, True),
                                                           (False, None, None, 9.0, False), (False, None, None, 9.0, True)])
def test_many_rows(ctx, causal, docs, prefix, cap, slopes, dtype):
    say(causal, docs, prefix, cap, slopes, dtype)
    Call(ctx, 650, causal=causal, docs=docs, prefix=prefix, cap=cap, slopes=slopes, dtype=dtype, **MANY).check()


# tiles that keep to their documents (128 rows or more on average), of any order of lengths, and tiles that cross them
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("docs,prefix", [([[200, 350]], None), ([[129, 0, 500, 1]], None), ([[33, 64, 500]], None), ([[650]], [[70]]), ([[1, 649]], [[1, 400]]), ([[128, 256, 256]], None),
                                         ([[5] * 130], None), ([[10] * 65], None), ([[9] * 63], [[i % 11 for i in range(63)]]), ([[0, 0, 0, 640]], None)])
def test_many_rows_of_documents(ctx, docs, prefix, causal):
    say(len(docs[0]), docs[0][:5], causal)
    prefix = prefix if causal else None  # (a prefix is causal)
    Call(ctx, 650, causal=causal, docs=docs, prefix=prefix, **MANY).check()
    Call(ctx, 650, causal=causal, docs=docs, prefix=prefix, slopes=True, **MANY).check()


def test_many_rows_of_documents_with_other_keys(ctx):
    Call(ctx, 650, 900, causal=False, docs=[[200, 350]], key_docs=[[0, 700]], **MANY).check()
    Call(ctx, 650, 300, causal=True, docs=[[200, 350]], key_docs=[[290, 10]], **MANY).check()
    Call(ctx, 330, batch=2, causal=True, docs=[[130, 200], [0, 300]], **MANY).check()


# few key blocks of a workgroup whose waves share them: fewer than its ring holds, whole and ragged
@pytest.mark.parametrize("keys", [1, 31, 32, 33, 64, 65, 97, 128, 129, 160, 161])
def test_few_key_blocks_of_many_rows(ctx, keys):
    say(keys)
    Call(ctx, 40, keys, batch=48, heads=12, kv=12, causal=False).check()
    Call(ctx, 40, keys, batch=48, heads=24, kv=12, causal=True, slopes=True).check()


# many rows over many keys: parts of 128-row tiles
def test_parts_of_many_rows(ctx):
    c = Call(ctx, 128, 8200, heads=8, kv=2, batch=2, causal=True)
    assert hip.lib().zdraw_hip_attention_masked_workspace(ctx.queue, C.byref(c.p)) > 128 * 8 * 2 * 130 * 4
    c.check()
    Call(ctx, 200, 17000, heads=6, kv=2, causal=False, cap=30.0).check()


# documents of no, one and many rows, more than a tile holds, rows behind the last; with other numbers of keys; padded segments
# a few tiles more than the GPU has units: the last ones are split along their keys, the others write their rows themselves
@pytest.mark.parametrize("causal,cap,slopes,dtype", [(False, 0.0, False, hip.BF16), (True, 0.0, False, hip.F16), (False, 9.0, False, hip.F16), (True, 0.0, True, hip.BF16), (True, 20.0, True, hip.BF16)])
@pytest.mark.parametrize("q,heads,kv", [(600, 52, 52), (299, 108, 54)])
def test_split_tail(ctx, q, heads, kv, causal, cap, slopes, dtype):
    say(q, heads, kv, causal, cap, slopes, dtype)
    L = hip.lib()
    c = Call(ctx, q, 2750, heads=heads, kv=kv, causal=causal, cap=cap, slopes=slopes, dtype=dtype, pad=(8, 0, 16))
    d = L.zdraw_hip_dispatch_count()
    n = L.zdraw_hip_attention_masked_workspace(ctx.queue, C.byref(c.p))
    assert 0 < n <= 14 * 5 * 128 * 130 * 4  # 4 or 14 tiles of 260 or 270, five shares at most
    first = c.check()
    assert L.zdraw_hip_dispatch_count() - d == 2
    room = ctx.buffer(np.full(n, 0xFF, np.uint8))
    c.o.workspace = room.handle
    c.clear()
    assert np.array_equal(c.check("workspace"), first)
    small = ctx.buffer(np.zeros(n - 16, np.uint8))
    c.o.workspace = small.handle
    assert c.rc() == hip.INVALID and "workspace" in hip.last_error()


# ... where rows of a split tile meet numbers that are not finite, in one share or in several
def test_split_tail_of_rows_that_meet_numbers_that_are_not_finite(ctx):
    def plant(c):
        inf = rr.bits(np.array([np.inf, -np.inf, np.nan], np.float32), c.dtype)
        for h in (47, 51):
            c.v[0, 20, h, 5] = inf[0]
            c.v[0, 2100, h, 6] = inf[1]
            c.k[0, 2190, h, 3] = inf[2]  # seen from row 40 on
        c.q[0, 10, 51, 3] = inf[2]

    c = Call(ctx, 600, 2750, heads=52, kv=52, x=plant)
    want, _, _ = c.want()
    assert np.isinf(want).any() and np.isnan(want).any()
    c.check()


def test_replayed_split_tail(ctx):
    L = hip.lib()
    c = Call(ctx, 600, 2100, heads=52, kv=52, causal=False)
    other = Call(ctx, 1, 60000, heads=8, kv=2, seed=5)
    queue = L.zdraw_hip_create_queue(ctx.device)
    first = c.check()
    keep = ctx.buffer(nbytes=L.zdraw_hip_attention_masked_workspace(queue, C.byref(c.p)))
    for room in (None, keep.handle):
        c.o.workspace = room
        g = rr.Captured(queue, c.enqueue)
        assert g.nodes() == (2 if room else 1)
        for _ in range(3):
            c.clear()
            g.replay()
            bits = c.check("replayed", run=False) if room is None else c.read()
            assert room is None or np.array_equal(bits, first)
            assert other.rc(queue) == 0
        g.close()
    L.zdraw_hip_release_queue(queue)


@pytest.mark.parametrize("docs,key_docs,batch,q,k", [
    ([[5, 0, 1, 40, 100]], None, 1, 150, 150), ([[1] * 70], None, 1, 70, 70), ([[0, 0]], None, 1, 9, 9), ([[10, 0, 20]], [[3, 5, 0]], 1, 64, 8),
    ([[7, 30]], [[300, 20]], 1, 37, 330), ([[1], [64], [17]], None, 3, 64, 64), ([[100, 28], [0, 77]], [[4, 200], [50, 60]], 2, 128, 260)])
@pytest.mark.parametrize("causal", [True, False])
def test_documents(ctx, docs, key_docs, batch, q, k, causal):
    say(docs, key_docs, causal)
    Call(ctx, q, k, batch=batch, heads=4, kv=2, causal=causal, docs=docs, key_docs=key_docs).check()


@pytest.mark.parametrize("prefix", [0, 1, 40, 100, 4000000000])
def test_prefix(ctx, prefix):
    class Held(Call):
        def want(self):
            self.prefix = np.minimum(self.prefix, self.kshape[1])
            return super().want()

    Held(ctx, 60, 100, prefix=[[prefix]]).check()


# cap and bias, alone and together, in every form that the rows take
@pytest.mark.parametrize("dtype", [hip.BF16, hip.F16])
@pytest.mark.parametrize("cap,slopes,causal", [(5.0, False, True), (50.0, False, False), (0.0, True, True), (0.0, True, False), (3.0, True, False)])
@pytest.mark.parametrize("q,k", [(1, 300), (70, 70)])
def test_cap_and_bias(ctx, q, k, cap, slopes, causal, dtype):
    say(q, k, cap, slopes, causal, dtype)
    Call(ctx, q, k, heads=6, kv=2, causal=causal, cap=cap, slopes=slopes, dtype=dtype, loud=3.0).check(scores=96.0)


@pytest.mark.parametrize("scale", [0.02, 1.0])
def test_scale(ctx, scale):
    Call(ctx, 50, scale=scale).check(scores=32.0 * scale * 11.4)


# rows with gaps between them, offsets, keys that all segments or heads share (stride 0)
def test_strides(ctx):
    Call(ctx, 45, 61, batch=2, heads=4, kv=2, pad=(16, 24, 40), off=24).check()
    c = Call(ctx, 45, 61, batch=2, heads=4, kv=2)
    for s in (c.p.k_stride, c.p.v_stride):
        s[0] = 0  # the first segment's keys
    c.k[1], c.v[1] = c.k[0], c.v[0]
    c.check("segments share keys")
    c = Call(ctx, 45, 61, heads=4, kv=2)
    c.p.k_stride[2] = 0
    c.k[:, :, 1] = c.k[:, :, 0]
    c.check("heads share keys")


# keys whose scores rise by far more than the room above the reference point, in the middle and at the end; and fall
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("q,heads", [(3, 2), (40, 56), (200, 2)])
def test_rising_scores(ctx, q, heads, sign):
    def climb(c):
        c.q[...] = rr.bits(np.full(c.shape, 1.0), c.dtype)
        steps = np.arange(c.kshape[1], dtype=np.float32)[None, :, None, None] * np.ones(c.kshape, np.float32)
        c.k[...] = rr.bits(sign * (steps // 16 * 0.5 - 20.0), c.dtype)

    Call(ctx, q, 900, heads=heads, kv=heads, causal=False, x=climb).check(scores=40.0 * 11.4)


# what a row does not see may hold anything: later keys, other documents', keys behind the last one, memory behind the keys
@pytest.mark.parametrize("dtype", [hip.BF16, hip.F16])
@pytest.mark.parametrize("heads", [2, 120, 240])
@pytest.mark.parametrize("nan", [float("nan"), float("inf"), -65504.0])
def test_unseen_keys_hold_anything(ctx, nan, heads, dtype):
    say(nan, heads, dtype)

    def rotten(c):
        c.k[0, 70:, :] = rr.bits(np.full_like(c.k[0, 70:], nan, np.float32), dtype)
        c.v[0, 70:, :] = rr.bits(np.full_like(c.v[0, 70:], nan, np.float32), dtype)

    c = Call(ctx, 150, heads=heads, kv=2, docs=[[70, 40]], causal=True, x=rotten, dtype=dtype)
    assert c.rc() == 0
    got = c.read()
    want, absolute, _ = c.want()
    rr.check(rr.value(got[0, :70], dtype), want[0, :70], absolute[0, :70], dtype, "the clean document")


def test_numbers_that_are_not_finite_reach_the_rows_that_see_them(ctx):
    def plant(c):
        inf = rr.bits(np.array([np.inf, -np.inf, np.nan], np.float32), c.dtype)
        c.v[0, 20, 0, 5] = inf[0]
        c.v[0, 33, 0, 6] = inf[1]
        c.v[0, 34, 1, 7] = inf[2]
        c.k[0, 40, 0, 3] = inf[2]
        c.q[0, 10, 1, 3] = inf[2]

    for q, heads, kv in ((50, 2, 2), (50, 90, 2), (600, 60, 60)):
        c = Call(ctx, q, heads=heads, kv=kv, x=plant)
        want, _, _ = c.want()
        assert np.isinf(want).any() and np.isnan(want).any()
        c.check()


def test_infinite_scores(ctx):
    def plant(c):
        c.q[0, 8] = rr.bits(np.full(c.q[0, 8].shape, 1e30), c.dtype)
        c.k[0, 0] = rr.bits(np.full(c.k[0, 0].shape, -1e30), c.dtype)  # -infinity for row 8 alone
        c.q[0, 0] = rr.bits(np.full(c.q[0, 0].shape, 1e30), c.dtype)   # a row whose only score is -infinity

    c = Call(ctx, 8 + 1, heads=2, kv=1, x=plant, causal=True)
    got = c.read() if c.rc() == 0 else None
    assert (got[0, 0] == 0).all()  # no weight anywhere: zeros, as without keys


# a call over few rows is split along its keys: through the queue's slots or a workspace the same bits; a graph holds no slot
def test_parts_and_workspace(ctx):
    L = hip.lib()
    c = Call(ctx, 2, 9000, heads=8, kv=2)
    n = L.zdraw_hip_attention_masked_workspace(ctx.queue, C.byref(c.p))
    assert n > 0
    first = c.check()
    again = c.check()
    assert np.array_equal(first, again)
    room = ctx.buffer(np.full(n, 0xFF, np.uint8))
    c.o.workspace = room.handle
    c.clear()
    assert np.array_equal(c.check("workspace"), first)
    small = ctx.buffer(np.zeros(n - 16, np.uint8))
    c.o.workspace = small.handle
    assert c.rc() == hip.INVALID and "workspace" in hip.last_error()


@pytest.mark.parametrize("room", [False, True])
def test_replayed_graph(ctx, room):
    L = hip.lib()
    c = Call(ctx, 2, 3000, heads=8, kv=2)
    other = Call(ctx, 1, 60000, heads=8, kv=2, seed=5)
    queue = L.zdraw_hip_create_queue(ctx.device)
    if room:
        keep = ctx.buffer(nbytes=L.zdraw_hip_attention_masked_workspace(queue, C.byref(c.p)))
        c.o.workspace = keep.handle
    g = rr.Captured(queue, c.enqueue)
    assert g.nodes() == (2 if room else 1)
    for _ in range(3):
        c.clear()
        g.replay()
        bits = c.check("replayed", run=False)
        assert other.rc(queue) == 0  # the queue's slots grow and are used meanwhile
        if room:
            c.clear()
            assert np.array_equal(c.check("eager"), bits)
    g.close()
    L.zdraw_hip_release_queue(queue)


def test_two_queues_at_once(ctx):
    L = hip.lib()
    calls = [Call(ctx, 1, 4000 + 100 * i, heads=8, kv=2, seed=i) for i in range(2)]
    queues = [L.zdraw_hip_create_queue(ctx.device) for _ in calls]
    batches = [L.zdraw_hip_batch_begin(q) for q in queues]
    for _ in range(5):
        for c, b in zip(calls, batches):
            assert c.enqueue(b) == 0
    for b in batches:
        assert L.zdraw_hip_batch_end(b) == 0
    for c in calls:
        c.check(run=False)
    for q in queues:
        L.zdraw_hip_release_queue(q)


# one head's keys span more than 4 GiB: the last of 20 keys, 2^28 - 128 bytes apart
def test_offsets_past_32_bits(ctx):
    keys, step = 20, (1 << 27) - 64  # elements
    c = Call(ctx, 3, keys, heads=2, kv=1, causal=False)
    span = ctx.buffer(nbytes=2 * ((keys - 1) * step + D))
    ptr = hip.lib().zdraw_hip_buffer_device_ptr(span.handle)
    piece = []
    for j in range(keys):
        h = hip.lib().zdraw_hip_wrap_device_memory(ctx.device, ptr + 2 * j * step, 2 * D)
        hip.lib().zdraw_hip_write_buffer(h, np.ascontiguousarray(c.k[0, j, 0]).ctypes.data_as(C.c_void_p), 2 * D)
        piece.append(h)
    c.bufs[1] = span
    c.p.k_stride[1] = step
    c.check()
    for h in piece:
        hip.lib().zdraw_hip_release_buffer(h)


def test_malformed_borders_stay_in_bounds(ctx):
    # borders past the segment and out of order: any rows, but only rows of the output, and no fault
    for borders in ([0, 500, 400, 4000000000], [90, 10, 80, 20], [4294967295] * 4, [0, 0, 0, 4294967295]):
        c = Call(ctx, 100, docs=[[30, 30, 40]])
        b = ctx.buffer(np.array(borders, np.uint32))
        c.o.q_starts = b.handle
        assert c.rc() == 0
        c.read()


def test_nothing_to_do(ctx):
    L = hip.lib()
    for field in ("q_tokens", "batch"):
        c = Call(ctx, 4)
        setattr(c.p, field, 0)
        d = L.zdraw_hip_dispatch_count()
        assert c.rc() == 0 and L.zdraw_hip_dispatch_count() == d
        assert (c.read() == POISON).all()
    c = Call(ctx, 4, 0)
    assert L.zdraw_hip_run_attention_masked(ctx.queue, c.bufs[0].handle, None, None, c.out.handle, C.byref(c.p), None) == 0
    assert (c.read() == 0).all()


@pytest.mark.parametrize("change,rc", [
    ({"head_dim": 64}, 1), ({"dtype": hip.F32}, 1), ({"heads": 0}, 2), ({"kv_heads": 3}, 2), ({"kv_heads": 0}, 2), ({"dtype": 9}, 2), ({"causal": 2}, 2),
    ({"scale": -1.0}, 2), ({"scale": float("nan")}, 2), ({"softcap": -1.0}, 2), ({"softcap": float("inf")}, 2), ({"reserved": 1}, 2), ({"q_tokens": 1 << 24}, 1),
    ({"k_tokens": 1 << 24}, 1), ({"q_tokens": 9}, 2), ({"k_tokens": 9}, 2), ({"batch": 2}, 2), ({"documents": 1}, 2), ({"q_off": 8}, 2), ({"out_off": 1 << 40}, 2),
    ({"q_stride": 4}, 2), ({"out_stride": 64}, 2), ({"k_stride": 1 << 60}, 2), ({"out_stride": 0}, 2)])
def test_refusals(ctx, change, rc):
    c = Call(ctx, 8, 8)
    for name, x in change.items():
        if name.endswith("stride"):
            getattr(c.p, name)[1] = x
        else:
            setattr(c.p, name, x)
    d = hip.lib().zdraw_hip_dispatch_count()
    assert c.rc() == rc, hip.last_error()
    assert hip.lib().zdraw_hip_dispatch_count() == d and hip.last_error()
    assert (c.out.read(np.uint16, c.size) == POISON).all()


def test_refused_operands(ctx):
    L = hip.lib()
    two = ctx.buffer(np.zeros(2, np.uint32))
    for change in ({"q_starts": two.handle}, {"k_starts": two.handle}, {"prefix": None}, {"slopes": two.handle}):
        c = Call(ctx, 8, causal=True)
        for name, x in change.items():
            if name == "prefix":
                c.p.causal, x = 0, two.handle
            setattr(c.o, name, x)
        assert c.rc() == 2, change
    c = Call(ctx, 8, 9, docs=[[8]], key_docs=[[9]])
    c.o.k_starts = None
    assert c.rc() == 2  # the queries' borders cannot stand for the keys'
    for i in range(3):
        c = Call(ctx, 8)
        args = list(c.args())
        args[i] = None
        assert L.zdraw_hip_run_attention_masked(ctx.queue, *args) == 2
    c = Call(ctx, 8)
    assert L.zdraw_hip_run_attention_masked(None, *c.args()) == -1
    assert L.zdraw_hip_run_attention_masked_enc(None, *c.args()) == -1
    assert L.zdraw_hip_run_attention_masked(ctx.queue, *c.args()[:4], None, None) == -1
