"""Attention of a batch over a shared prefix (zdraw_hip_run_attention_shared), the cache append (zdraw_hip_run_kv_append) and the
two together, against their definitions in 64 bits. Tolerances count roundings (tests/rangeref.py)."""
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


def say(*a):
    print(*a, flush=True)


class Shared:
    def __init__(self, ctx, requests, q=1, prefix=0, capacity=0, *, lens=None, q_lens=None, page=0, heads=4, kv=2, causal=True, cap=0.0, slopes=False,
                 dtype=hip.BF16, pad=(0, 0, 0), seed=0, table=None, pool=None):
        self.ctx, self.dtype, self.causal, self.cap, self.page, self.capacity, self.prefix = ctx, dtype, causal, cap, page, capacity, prefix
        rng = np.random.default_rng(seed + requests + 3 * q + prefix + capacity)
        draw = lambda s, c=1.0: rr.bits(rng.standard_normal(s, dtype=np.float32) * c, dtype)
        self.shape = (requests, q, heads, D)
        self.q = draw(self.shape, 1.2)
        self.pk, self.pv = draw((1, prefix, kv, D)), draw((1, prefix, kv, D))
        self.lens = np.array([capacity] * requests if lens is None else lens, np.uint32)
        self.q_lens = None if q_lens is None else np.array(q_lens, np.uint32)
        self.slopes = np.float32(2.0) ** -np.arange(1, heads + 1, dtype=np.float32) if slopes else None
        self.per = -(-capacity // page) if page else 0
        if page:
            pool = pool or requests * self.per + 2
            self.table = np.array(rng.permutation(pool)[:requests * self.per].reshape(requests, self.per) if table is None else table, np.uint32)
            kshape = (pool, page, kv, D)
        else:
            self.table = None
            kshape = (requests, capacity, kv, D)
        self.k, self.v = np.full(kshape, POISON, np.uint16), np.full(kshape, POISON, np.uint16)
        for r in range(requests):  # keys past a request's length, pages that nobody has: NaN
            for j in range(min(int(self.lens[r]), capacity)):
                at = self.place(r, j)
                self.k[at], self.v[at] = draw((kv, D)), draw((kv, D))
        p, o = hip.SharedAttn(), hip.SharedOperands()
        p.requests, p.q_tokens, p.prefix_tokens, p.capacity, p.page_tokens, p.pages = requests, q, prefix, capacity, page, kshape[0] if page else 0
        p.heads, p.kv_heads, p.head_dim, p.dtype, p.causal, p.softcap = heads, kv, D, dtype, int(causal), cap
        self.p, self.o, self.keep = p, o, []

        def put(x, strides):
            size = rr.dense(strides, x.shape, pad)
            self.keep.append(ctx.buffer(np.concatenate((rr.spread(x, strides, size, np.uint16(POISON)), np.full(8, POISON, np.uint16)))))
            return self.keep[-1].handle

        pks, pvs = (C.c_uint64 * 3)(), (C.c_uint64 * 3)()
        self.handles = [put(self.q, p.q_stride), put(self.pk, pks), put(self.pv, pvs), put(self.k, p.k_stride), put(self.v, p.v_stride)]
        p.prefix_k_stride[0], p.prefix_k_stride[1], p.prefix_v_stride[0], p.prefix_v_stride[1] = pks[1], pks[2], pvs[1], pvs[2]
        self.size = rr.dense(p.out_stride, self.shape, pad)
        self.out = ctx.buffer(np.full(self.size, POISON, np.uint16))
        for name, a in (("lens", self.lens), ("q_lens", self.q_lens), ("page_table", self.table), ("slopes", self.slopes)):
            if a is not None and a.size:
                self.keep.append(ctx.buffer(a))
                setattr(o, name, self.keep[-1].handle)

    def place(self, r, j):
        if not self.page:
            return r, j
        return min(int(self.table[r, j // self.page]), self.k.shape[0] - 1), j % self.page

    def args(self):
        return (*self.handles, self.out.handle, C.byref(self.p), C.byref(self.o))

    def rc(self, queue=None):
        return hip.lib().zdraw_hip_run_attention_shared(queue or self.ctx.queue, *self.args())

    def enqueue(self, batch):
        return hip.lib().zdraw_hip_run_attention_shared_enc(batch, *self.args())

    def clear(self):
        self.out.write(np.full(self.size, POISON, np.uint16))

    def check(self, what="", run=True, scores=32.0):
        if run:
            rc = self.rc()
            assert rc == 0, hip.last_error()
        flat = self.out.read(np.uint16, self.size)
        got = rr.gather(flat, self.p.out_stride, self.shape)
        mask = rr.spread(np.ones(self.shape, np.uint16), self.p.out_stride, self.size, np.uint16(0))
        assert (flat[mask == 0] == POISON).all()
        f = lambda b: rr.value(b, self.dtype)
        requests, q, heads, _ = self.shape
        for r in range(requests):
            n = min(int(self.lens[r]), self.capacity)
            ql = q if self.q_lens is None else min(int(self.q_lens[r]), q)
            own = [self.place(r, j) for j in range(n)]
            kv = self.k.shape[2]
            cat = lambda pre, x: np.concatenate([f(pre[0]), f(np.array([x[at] for at in own], np.uint16).reshape(n, kv, D))])
            at = self.prefix + n - ql + np.arange(ql)
            j = np.arange(self.prefix + n)
            seen = np.ones((ql, self.prefix + n), bool) if not self.causal else (j[None] < self.prefix) | (j[None] <= at[:, None])
            want, absolute = rr.rows(f(self.q[r, :ql]), cat(self.pk, self.k), cat(self.pv, self.v), seen, at, 0.0, self.cap, self.slopes)
            rr.check(f(got[r, :ql]), want, absolute, self.dtype, f"{what} request {r}", scores)
            assert (got[r, ql:] == POISON).all(), f"request {r}: rows past its own were written"
        return got


@pytest.mark.parametrize("dtype", [hip.BF16, hip.F16])
@pytest.mark.parametrize("requests,q,prefix,capacity,page,heads,kv", [
    (1, 1, 1, 1, 0, 1, 1), (3, 1, 100, 50, 0, 4, 2), (5, 1, 33, 70, 16, 8, 1), (40, 1, 300, 40, 4, 4, 2), (2, 3, 257, 31, 8, 16, 2), (9, 5, 64, 96, 32, 6, 3),
    (1, 40, 500, 60, 64, 2, 2), (3, 70, 90, 130, 16, 2, 1), (2, 1, 3000, 700, 256, 4, 4)])
def test_requests_over_a_prefix(ctx, requests, q, prefix, capacity, page, heads, kv, dtype):
    say(requests, q, prefix, capacity, page, heads, kv, dtype)
    lens = [max(q, capacity - 7 * r) if capacity >= q else capacity for r in range(requests)]
    Shared(ctx, requests, q, prefix, capacity, lens=lens, page=page, heads=heads, kv=kv, dtype=dtype).check()


# rows that fill workgroups by themselves: they walk the prefix, then their own keys
@pytest.mark.parametrize("page", [0, 4, 8, 16, 64])
@pytest.mark.parametrize("causal,cap,slopes", [(True, 0.0, False), (False, 0.0, False), (True, 12.0, True), (False, 0.0, True)])
def test_many_rows_walk_both(ctx, causal, cap, slopes, page):
    d = hip.lib().zdraw_hip_dispatch_count()
    Shared(ctx, 3, 140, 200, 150, lens=[150, 140, 141], page=page, heads=32, kv=32, causal=causal, cap=cap, slopes=slopes).check()
    assert hip.lib().zdraw_hip_dispatch_count() - d == 1
    Shared(ctx, 4, 700, 130, 720, lens=[0, 700, 33, 719], q_lens=[5, 700, 0, 699], page=page, heads=16, kv=16, causal=causal, cap=cap, slopes=slopes).check()


# a few workgroups over the GPU's units, or half of its units: the last ones' prefix and own keys are split (and 66 rows of 128
# workgroups are few enough for the form whose waves take the key blocks in turn)
@pytest.mark.parametrize("causal,cap,slopes", [(False, 0.0, False), (True, 0.0, False), (True, 12.0, True)])
@pytest.mark.parametrize("requests,q,kv,page,lens,q_lens", [
    (2, 66, 64, 0, [200, 131], None), (2, 127, 64, 0, [200, 131], None), (3, 66, 86, 16, [0, 200, 77], [66, 40, 66]),
    (4, 66, 65, 64, [200, 64, 65, 4000000000], [0, 66, 1, 66])])
def test_split_tail(ctx, requests, q, kv, page, lens, q_lens, causal, cap, slopes):
    say(requests, q, kv, page, lens, causal, cap, slopes)
    c = Shared(ctx, requests, q, 2100, 200, lens=lens, q_lens=q_lens, page=page, heads=kv, kv=kv, causal=causal, cap=cap, slopes=slopes)
    split = (requests, q) != (2, 66)
    n = hip.lib().zdraw_hip_attention_shared_workspace(ctx.queue, C.byref(c.p))
    assert (n > 0) == split
    d = hip.lib().zdraw_hip_dispatch_count()
    first = c.check()
    assert hip.lib().zdraw_hip_dispatch_count() - d == 1 + split
    room = ctx.buffer(np.full(max(n, 16), 0xFF, np.uint8))
    c.o.workspace = room.handle
    c.clear()
    assert np.array_equal(c.check("workspace"), first)


# the prefix for many requests at once through the form whose waves share key blocks: a launch of its own
@pytest.mark.parametrize("slopes", [False, True])
def test_rows_of_many_requests_share_key_blocks(ctx, slopes):
    d = hip.lib().zdraw_hip_dispatch_count()
    Shared(ctx, 70, 1, 24000, 20, lens=[(7 * r) % 21 for r in range(70)], q_lens=[r % 3 != 1 for r in range(70)], page=4, heads=32, kv=1, slopes=slopes).check()
    assert hip.lib().zdraw_hip_dispatch_count() - d == 3  # the prefix, the requests' own keys, the join


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("prefix,capacity,lens,q_lens", [
    (0, 40, [40, 0, 3, 17], None), (50, 0, [0, 0, 0, 0], None), (0, 0, [0] * 4, None), (20, 30, [0, 1, 30, 4000000000], None),
    (20, 30, [5, 6, 7, 8], [0, 1, 2, 4000000000]), (0, 30, [1, 0, 30, 2], [2, 2, 1, 0])])
def test_lengths(ctx, prefix, capacity, lens, q_lens, causal):
    say(prefix, capacity, lens, q_lens)
    for page in (0, 8) if capacity else (0,):
        Shared(ctx, 4, 2, prefix, capacity, lens=lens, q_lens=q_lens, page=page, causal=causal).check(f"page {page}")


@pytest.mark.parametrize("cap,slopes", [(4.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("q", [1, 90])
def test_cap_and_bias_count_the_prefix(ctx, q, cap, slopes):
    Shared(ctx, 2, q, 130, 100, lens=[100, 93], page=16, heads=4, kv=2, cap=cap, slopes=slopes).check()


def test_strides(ctx):
    Shared(ctx, 3, 2, 40, 50, lens=[50, 2, 33], page=16, pad=(8, 16, 32)).check()
    Shared(ctx, 3, 2, 40, 50, lens=[50, 2, 33], pad=(8, 16, 32)).check()


# two requests on the same pages, one page for all of a request's keys, pages past the pool (held to its last page)
def test_pages_in_any_order(ctx):
    Shared(ctx, 2, 1, 10, 32, page=16, table=[[3, 1], [3, 1]], pool=4, lens=[32, 32]).check()
    Shared(ctx, 2, 1, 10, 32, page=16, table=[[1, 1], [0, 0]], pool=2, lens=[32, 20]).check()
    Shared(ctx, 2, 1, 10, 32, page=16, table=[[1, 4000000000], [0, 5]], pool=5, lens=[32, 20]).check()
    # past a request's length nothing is looked up
    Shared(ctx, 2, 1, 10, 64, page=16, table=[[1, 0xFFFFFFFF, 0xFFFFFFFF, 0xFFFFFFFF], [0, 2, 0xFFFFFFFF, 0xFFFFFFFF]], pool=3, lens=[16, 17]).check()


def test_workspace_and_graph(ctx):
    L = hip.lib()
    c = Shared(ctx, 6, 1, 700, 90, lens=[90, 1, 33, 64, 65, 12], page=16, heads=8, kv=2)
    first = c.check()
    n = L.zdraw_hip_attention_shared_workspace(ctx.queue, C.byref(c.p))
    assert n > 0
    room = ctx.buffer(np.full(n, 0xFF, np.uint8))
    queue = L.zdraw_hip_create_queue(ctx.device)
    for handle in (None, room.handle):
        c.o.workspace = handle
        g = rr.Captured(queue, c.enqueue)
        assert g.nodes() == (2 if handle else 1)  # without a workspace unsplit: a graph holds no slot
        for _ in range(3):
            c.clear()
            g.replay()
            bits = c.check("replayed", run=False)
            if handle:
                assert np.array_equal(bits, first)
            assert Shared(ctx, 20, 1, 2000, 64, page=16, heads=8, kv=2).rc(queue) == 0
        g.close()
    L.zdraw_hip_release_queue(queue)
    small = ctx.buffer(np.zeros(n - 16, np.uint8))
    c.o.workspace = small.handle
    assert c.rc() == hip.INVALID


def test_nothing_to_do(ctx):
    for field in ("requests", "q_tokens"):
        c = Shared(ctx, 2, 1, 10, 10)
        setattr(c.p, field, 0)
        d = hip.lib().zdraw_hip_dispatch_count()
        assert c.rc() == 0 and hip.lib().zdraw_hip_dispatch_count() == d
        assert (c.out.read(np.uint16, c.size) == POISON).all()


@pytest.mark.parametrize("change,rc", [
    ({"head_dim": 64}, 1), ({"dtype": hip.F32}, 1), ({"heads": 3}, 2), ({"dtype": 7}, 2), ({"causal": 2}, 2), ({"scale": float("inf")}, 2), ({"softcap": -2.0}, 2),
    ({"reserved": 9}, 2), ({"page_tokens": 24}, 2), ({"page_tokens": 2}, 1), ({"pages": 0}, 2), ({"pages": 99}, 2), ({"capacity": 90}, 2), ({"requests": 9}, 2),
    ({"prefix_tokens": 41}, 2), ({"prefix_tokens": 1 << 24}, 1), ({"q_off": 2}, 2), ({"prefix_v_off": 1 << 50}, 2), ({"k_stride": 4}, 2), ({"out_stride": 0}, 2)])
def test_refusals(ctx, change, rc):
    c = Shared(ctx, 3, 2, 40, 32, page=16)
    for name, x in change.items():
        if name.endswith("stride"):
            getattr(c.p, name)[1] = x
        else:
            setattr(c.p, name, x)
    assert c.rc() == rc, hip.last_error()
    assert (c.out.read(np.uint16, c.size) == POISON).all()


def test_refused_operands(ctx):
    L = hip.lib()
    one = ctx.buffer(np.zeros(1, np.uint32))
    for name, x in (("lens", None), ("lens", one.handle), ("q_lens", one.handle), ("page_table", None), ("page_table", one.handle), ("slopes", one.handle)):
        c = Shared(ctx, 3, 2, 40, 32, page=16)
        setattr(c.o, name, x)
        assert c.rc() == 2, name
    c = Shared(ctx, 3, 2, 40, 32)
    c.o.page_table = one.handle
    assert c.rc() == 2  # a table without pages
    for i in range(6):
        c = Shared(ctx, 3, 2, 40, 32, page=16)
        args = list(c.args())
        args[i] = None
        assert L.zdraw_hip_run_attention_shared(ctx.queue, *args) == 2
    assert L.zdraw_hip_run_attention_shared(None, *c.args()) == -1
    assert L.zdraw_hip_run_attention_shared_enc(None, *c.args()) == -1
    assert L.zdraw_hip_run_attention_shared(ctx.queue, *c.args()[:7], None) == -1


# ------------------------------------------------------------------ cache append
class Append:
    def __init__(self, ctx, requests, tokens, capacity, *, starts, counts=None, page=0, heads=4, kv=2, act=hip.BF16, dtype=hip.BF16, rotation=hip.ROTATE_NONE,
                 norm=False, rope_rows=0, base=0, pad=(0, 0, 0), table=None, pool=None, seed=0, eps=1e-6):
        self.ctx, self.act, self.dtype, self.page, self.capacity, self.rotation, self.base = ctx, act, dtype, page, capacity, rotation, base
        rng = np.random.default_rng(seed + 11 * requests + tokens + capacity)
        self.qs, self.ks = (requests, tokens, heads, D), (requests, tokens, kv, D)
        draw = lambda s: rng.standard_normal(s, dtype=np.float32) * 2
        conv = (lambda x: x) if act == hip.F32 else (lambda x: rr.bits(x, act))
        self.q, self.k, self.v = conv(draw(self.qs)), conv(draw(self.ks)), conv(draw(self.ks))
        self.starts = np.array(starts, np.uint32)
        self.counts = None if counts is None else np.array(counts, np.uint32)
        self.per = -(-capacity // page) if page else 0
        if page:
            pool = pool or requests * self.per + 1
            self.table = np.array(rng.permutation(pool)[:requests * self.per].reshape(requests, self.per) if table is None else table, np.uint32)
            self.cs = (pool, page, kv, D)
        else:
            self.table, self.cs = None, (requests, capacity, kv, D)
        self.wq, self.wk = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)) if norm else (None, None)
        self.eps = eps
        if rotation:
            ang = rng.uniform(0, 6.28, (rope_rows, D // 2))
            ang = np.repeat(ang, 2, 1) if rotation == hip.ROTATE_PAIRS else np.concatenate((ang, ang), 1)
            self.cos, self.sin = np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)
        else:
            self.cos = self.sin = None
        p, o = hip.KvAppend(), hip.AppendOperands()
        p.requests, p.tokens, p.capacity, p.page_tokens, p.pages = requests, tokens, capacity, page, self.cs[0] if page else 0
        p.heads, p.kv_heads, p.head_dim, p.in_dtype, p.dtype, p.rotation, p.rope_rows, p.position_base, p.eps = heads, kv, D, act, dtype, rotation, rope_rows, base, eps
        self.p, self.o, self.keep, self.handles = p, o, [], []
        for x, dst in ((self.q, p.q_stride), (self.k, p.k_stride), (self.v, p.v_stride)):
            size = rr.dense(dst, x.shape, pad)
            self.keep.append(ctx.buffer(np.concatenate((rr.spread(x, dst, size, x.dtype.type(0)), np.zeros(8, x.dtype)))))
            self.handles.append(self.keep[-1].handle)
        self.outs = []
        for s, dst in ((self.qs, p.q_out_stride), (self.cs, p.cache_k_stride), (self.cs, p.cache_v_stride)):
            size = rr.dense(dst, s, pad)
            self.outs.append((ctx.buffer(np.full(size + 8, POISON, np.uint16)), dst, s, size))
            self.handles.append(self.outs[-1][0].handle)
        for name, a in (("starts", self.starts), ("counts", self.counts), ("page_table", self.table), ("q_weight", self.wq if heads else None), ("k_weight", self.wk),
                        ("rope_cos", self.cos), ("rope_sin", self.sin)):
            if a is not None:
                self.keep.append(ctx.buffer(a))
                setattr(o, name, self.keep[-1].handle)

    def args(self):
        return (*self.handles, C.byref(self.p), C.byref(self.o))

    def rc(self, queue=None):
        return hip.lib().zdraw_hip_run_kv_append(queue or self.ctx.queue, *self.args())

    def enqueue(self, batch):
        return hip.lib().zdraw_hip_run_kv_append_enc(batch, *self.args())

    def turned(self, x, w, pos):
        """One row [heads][D] in f64."""
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(self.eps))) * w.astype(np.float64)
        if not self.rotation:
            return x
        r = min(pos, self.cos.shape[0] - 1)
        c, s = self.cos[r].astype(np.float64), self.sin[r].astype(np.float64)
        o = np.empty_like(x)
        if self.rotation == hip.ROTATE_PAIRS:
            o[:, 0::2], o[:, 1::2] = -x[:, 1::2], x[:, 0::2]
        else:
            o[:, :64], o[:, 64:] = -x[:, 64:], x[:, :64]
        return x * c + o * s

    def check(self, run=True):
        if run:
            assert self.rc() == 0, hip.last_error()
        f = (lambda x: x.astype(np.float64)) if self.act == hip.F32 else (lambda x: rr.value(x, self.act))
        want = [np.full(s, np.nan) for s in (self.qs, self.cs, self.cs)]
        for r in range(self.qs[0]):
            n = self.qs[1] if self.counts is None else min(int(self.counts[r]), self.qs[1])
            for t in range(n):
                at = int(self.starts[r]) + t
                pos = at + self.base
                want[0][r, t] = self.turned(f(self.q[r, t]), self.wq, pos)
                if at >= self.capacity:
                    continue
                where = (r, at)
                if self.page:
                    where = (int(self.table[r, at // self.page]), at % self.page)
                    if where[0] >= self.cs[0]:
                        continue
                want[1][where], want[2][where] = self.turned(f(self.k[r, t]), self.wk, pos), f(self.v[r, t])
        for i, ((buf, strides, shape, size), w) in enumerate(zip(self.outs, want)):
            flat = buf.read(np.uint16, size + 8)
            got = rr.gather(flat, strides, shape)
            mask = rr.spread(np.ones(shape, np.uint16), strides, size, np.uint16(0))
            assert (flat[:size][mask == 0] == POISON).all() and (flat[size:] == POISON).all()
            still = np.isnan(w)
            assert (got[still] == POISON).all(), f"output {i}: places outside of the new rows were written"
            g, x = rr.value(got[~still], self.dtype), w[~still]
            # half a step of the type; f32 behind it: 128 squares, the reciprocal root, two products and a sum: 2^-24 each, of
            # numbers no larger than the row's largest
            big = np.abs(np.nan_to_num(w)).max(-1, keepdims=True) + np.zeros_like(w)
            allowed = rr.HALF[self.dtype] * np.abs(x) + 2.0 ** -24 * 140 * 1.5 * big[~still] + (2.0 ** -25 if self.dtype == hip.F16 else 0.0)
            err = np.abs(g - x)
            assert (err <= allowed).all(), f"output {i}: {err.max()} off, {(err / allowed).max()} of what is allowed"


@pytest.mark.parametrize("rotation", [hip.ROTATE_NONE, hip.ROTATE_PAIRS, hip.ROTATE_HALVES])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("act,dtype", [(hip.F32, hip.BF16), (hip.F32, hip.F16), (hip.BF16, hip.BF16), (hip.F16, hip.F16), (hip.BF16, hip.F16), (hip.F16, hip.BF16)])
def test_append(ctx, act, dtype, norm, rotation):
    say(act, dtype, norm, rotation)
    Append(ctx, 3, 5, 20, starts=[0, 7, 15], page=8, act=act, dtype=dtype, norm=norm, rotation=rotation, rope_rows=20).check()


@pytest.mark.parametrize("requests,tokens,capacity,page,heads,kv,starts,counts", [
    (1, 1, 1, 0, 1, 1, [0], None), (4, 1, 40, 16, 8, 2, [0, 15, 16, 39], None), (2, 70, 100, 0, 3, 3, [0, 30], [70, 1]), (3, 33, 64, 4, 0, 2, [0, 31, 5], [33, 0, 32]),
    (2, 700, 800, 64, 30, 10, [100, 0], [700, 650]), (2, 4, 8, 8, 2, 1, [6, 4294967295], None), (2, 4, 8, 0, 2, 1, [7, 9], [4000000000, 3])])
def test_append_places(ctx, requests, tokens, capacity, page, heads, kv, starts, counts):
    say(requests, tokens, capacity, page, heads, kv, starts, counts)
    Append(ctx, requests, tokens, capacity, page=page, heads=heads, kv=kv, starts=starts, counts=counts, norm=True, rotation=hip.ROTATE_HALVES, rope_rows=capacity).check()


def test_append_strides_positions_and_pages(ctx):
    Append(ctx, 2, 6, 30, starts=[3, 20], pad=(8, 16, 24), rotation=hip.ROTATE_PAIRS, rope_rows=30, norm=True).check()
    Append(ctx, 2, 6, 30, starts=[3, 20], page=16, pad=(8, 16, 24), act=hip.F32).check()
    Append(ctx, 2, 6, 30, starts=[3, 20], base=1000, rotation=hip.ROTATE_HALVES, rope_rows=1024).check()
    Append(ctx, 2, 6, 30, starts=[3, 20], base=4294967295, rotation=hip.ROTATE_HALVES, rope_rows=7).check()  # held to the last row
    Append(ctx, 2, 6, 32, starts=[12, 13], page=16, table=[[0, 4000000000], [1, 3]], pool=3).check()  # rows on pages that are not there are not kept


def test_append_leaves_values_that_are_not_finite_in_their_rows(ctx):
    c = Append(ctx, 1, 3, 8, starts=[2], norm=True, rotation=hip.ROTATE_HALVES, rope_rows=8)
    bad = c.k.copy()
    bad[0, 1, 0, 4] = rr.bits(np.array([np.inf], np.float32), hip.BF16)[0]
    hip.lib().zdraw_hip_write_buffer(c.handles[1], bad.ctypes.data_as(C.c_void_p), bad.nbytes)
    assert c.rc() == 0
    buf, strides, shape, size = c.outs[1]
    got = rr.value(rr.gather(buf.read(np.uint16, size + 8), strides, shape), hip.BF16)
    assert np.isnan(got[0, 3, 0]).any() and np.isfinite(got[0, 2]).all() and np.isfinite(got[0, 4]).all() and np.isfinite(got[0, 3, 1]).all()


@pytest.mark.parametrize("change,rc", [
    ({"head_dim": 64}, 1), ({"dtype": hip.F32}, 1), ({"dtype": 5}, 2), ({"in_dtype": 5}, 2), ({"rotation": 3}, 2), ({"eps": -1.0}, 2), ({"kv_heads": 0}, 2),
    ({"capacity": 0}, 2), ({"capacity": 1 << 24}, 1), ({"page_tokens": 12}, 2), ({"page_tokens": 1}, 1), ({"pages": 0}, 2), ({"pages": 99}, 2), ({"rope_rows": 0}, 2), ({"rope_rows": 99}, 2),
    ({"tokens": 9}, 2), ({"requests": 99}, 2), ({"heads": 0}, 2), ({"k_off": 8}, 2), ({"cache_v_stride": 0}, 2), ({"q_out_stride": 100}, 2)])
def test_append_refusals(ctx, change, rc):
    c = Append(ctx, 2, 6, 30, starts=[3, 20], page=16, norm=True, rotation=hip.ROTATE_HALVES, rope_rows=30)
    for name, x in change.items():
        if name.endswith("stride"):
            getattr(c.p, name)[1] = x
        else:
            setattr(c.p, name, x)
    assert c.rc() == rc, hip.last_error()
    for buf, _, _, size in c.outs:
        assert (buf.read(np.uint16, size + 8) == POISON).all()


def test_append_refused_operands(ctx):
    L = hip.lib()
    one = ctx.buffer(np.zeros(1, np.uint32))
    for name, x in (("starts", None), ("starts", one.handle), ("counts", one.handle), ("page_table", None), ("page_table", one.handle), ("q_weight", one.handle),
                    ("k_weight", one.handle), ("rope_cos", None), ("rope_sin", one.handle)):
        c = Append(ctx, 2, 6, 30, starts=[3, 20], page=16, norm=True, rotation=hip.ROTATE_HALVES, rope_rows=30)
        setattr(c.o, name, x)
        assert c.rc() == 2, name
    for i in range(6):
        args = list(Append(ctx, 2, 6, 30, starts=[3, 20]).args())
        args[i] = None
        assert L.zdraw_hip_run_kv_append(ctx.queue, *args) == 2
    c = Append(ctx, 2, 6, 30, starts=[3, 20])
    c.p.requests = 0
    assert c.rc() == 0
    c = Append(ctx, 2, 6, 30, starts=[3, 20])
    c.p.tokens = 0
    assert c.rc() == 0
    assert L.zdraw_hip_run_kv_append(None, *c.args()) == -1 and L.zdraw_hip_run_kv_append_enc(None, *c.args()) == -1
    assert L.zdraw_hip_run_kv_append(ctx.queue, *c.args()[:7], None) == -1


# ------------------------------------------------------------------ as they are used together
def test_prompt_then_tokens(ctx):
    """A prompt attends to itself (masked), its keys stay as the prefix; two requests then append and attend step by step,
    in one batch, and as a graph that is replayed."""
    L = hip.lib()
    heads, kv, prompt, steps, page, dt = 4, 2, 70, 3, 8, hip.BF16
    requests, capacity = 2, 16
    rng = np.random.default_rng(9)
    f = lambda x: rr.value(x, dt)
    draw = lambda *s: rr.bits(rng.standard_normal(s, dtype=np.float32), dt)
    rope_rows = prompt + capacity
    ang = np.arange(rope_rows)[:, None] * 10000.0 ** (-np.arange(64) / 64)
    ang = np.concatenate((ang, ang), 1)
    cos, sin = ctx.buffer(np.cos(ang).astype(np.float32)), ctx.buffer(np.sin(ang).astype(np.float32))
    queue = L.zdraw_hip_create_queue(ctx.device)

    def append(q, k, v, n, requests, starts, base, pages, table, capacity, qo, ck, cv):
        p, o = hip.KvAppend(), hip.AppendOperands()
        p.requests, p.tokens, p.capacity, p.page_tokens, p.pages = requests, n, capacity, page if table else 0, pages
        p.heads, p.kv_heads, p.head_dim, p.in_dtype, p.dtype, p.rotation, p.rope_rows, p.position_base = heads, kv, D, dt, dt, hip.ROTATE_HALVES, rope_rows, base
        for dst, c in ((p.q_stride, heads), (p.k_stride, kv), (p.v_stride, kv), (p.q_out_stride, heads)):
            rr.dense(dst, (requests, n, c, D))
        for dst in (p.cache_k_stride, p.cache_v_stride):
            rr.dense(dst, (pages or requests, page if table else capacity, kv, D))
        o.starts, o.rope_cos, o.rope_sin, o.page_table = starts.handle, cos.handle, sin.handle, table.handle if table else None
        return lambda b: L.zdraw_hip_run_kv_append_enc(b, q.handle, k.handle, v.handle, qo.handle, ck.handle, cv.handle, C.byref(p), C.byref(o))

    # the prompt: append into a plain cache, attend causally
    q0, k0, v0 = draw(1, prompt, heads, D), draw(1, prompt, kv, D), draw(1, prompt, kv, D)
    bufs = [ctx.buffer(x) for x in (q0, k0, v0)]
    qo, pk, pv, out0 = (ctx.buffer(nbytes=2 * prompt * n * D) for n in (heads, kv, kv, heads))
    zero = ctx.buffer(np.zeros(1, np.uint32))
    first = append(*bufs, prompt, 1, zero, 0, 0, None, prompt, qo, pk, pv)
    mp = hip.MaskedAttn()
    mp.batch, mp.q_tokens, mp.k_tokens, mp.heads, mp.kv_heads, mp.head_dim, mp.dtype, mp.causal = 1, prompt, prompt, heads, kv, D, dt, 1
    for dst, c in ((mp.q_stride, heads), (mp.k_stride, kv), (mp.v_stride, kv), (mp.out_stride, heads)):
        rr.dense(dst, (1, prompt, c, D))
    batch = L.zdraw_hip_batch_begin(queue)
    assert first(batch) == 0, hip.last_error()
    assert L.zdraw_hip_run_attention_masked_enc(batch, qo.handle, pk.handle, pv.handle, out0.handle, C.byref(mp), None) == 0, hip.last_error()

    # the steps
    per = capacity // page
    pool = requests * per
    table = np.array([[2, 0], [1, 3]], np.uint32)
    tb = ctx.buffer(table)
    ck, cv = ctx.buffer(np.full((pool, page, kv, D), POISON, np.uint16)), ctx.buffer(np.full((pool, page, kv, D), POISON, np.uint16))
    qs, ks, vs = draw(steps, requests, 1, heads, D), draw(steps, requests, 1, kv, D), draw(steps, requests, 1, kv, D)
    begin = np.array([6, 0], np.uint32)  # the first request's steps cross a page
    seeds = draw(6, kv, D), draw(6, kv, D)
    image = np.full((pool, page, kv, D), POISON, np.uint16)
    for i, b in enumerate((ck, cv)):
        x = image.copy()
        x[table[0, 0], :6] = seeds[i]
        b.write(x)
    outs, calls, keep = [], [], []
    for s in range(steps):
        sq, sk, sv = (ctx.buffer(x[s]) for x in (qs, ks, vs))
        starts, lens = ctx.buffer(begin + np.uint32(s)), ctx.buffer(begin + np.uint32(s + 1))
        sqo, so = (ctx.buffer(nbytes=2 * requests * heads * D) for _ in range(2))
        p, o = hip.SharedAttn(), hip.SharedOperands()
        p.requests, p.q_tokens, p.prefix_tokens, p.capacity, p.page_tokens, p.pages = requests, 1, prompt, capacity, page, pool
        p.heads, p.kv_heads, p.head_dim, p.dtype, p.causal = heads, kv, D, dt, 1
        for dst in (p.q_stride, p.out_stride):
            rr.dense(dst, (requests, 1, heads, D))
        for dst in (p.k_stride, p.v_stride):
            rr.dense(dst, (pool, page, kv, D))
        for dst in (p.prefix_k_stride, p.prefix_v_stride):
            dst[0], dst[1] = kv * D, D
        o.lens, o.page_table = lens.handle, tb.handle
        room = ctx.buffer(nbytes=max(16, L.zdraw_hip_attention_shared_workspace(queue, C.byref(p))))
        o.workspace = room.handle
        put = append(sq, sk, sv, 1, requests, starts, prompt, pool, tb, capacity, sqo, ck, cv)
        args = (sqo.handle, pk.handle, pv.handle, ck.handle, cv.handle, so.handle, C.byref(p), C.byref(o))
        calls.append((put, args))
        outs.append(so)
        keep += [sq, sk, sv, starts, lens, sqo, room, p, o]

    def all_steps(b):
        for put, args in calls:
            rc = put(b)
            if rc == 0:
                rc = L.zdraw_hip_run_attention_shared_enc(b, *args)
            if rc:
                return rc
        return 0

    assert all_steps(batch) == 0, hip.last_error()
    assert L.zdraw_hip_batch_end(batch) == 0

    # the same by the definition, from the rotated and rounded rows
    def turn(x, pos):
        c, s = np.cos(ang[pos]).astype(np.float32).astype(np.float64), np.sin(ang[pos]).astype(np.float32).astype(np.float64)
        y = np.concatenate((-x[..., 64:], x[..., :64]), -1)
        return x * c + y * s

    kp = np.stack([turn(f(k0[0, t]), t) for t in range(prompt)])
    got_k = f(pk.read(np.uint16, (prompt, kv, D)))
    assert (np.abs(got_k - kp) <= rr.HALF[dt] * np.abs(kp) + 2.0 ** -20).all()
    qp = f(qo.read(np.uint16, (prompt, heads, D)))
    pos = np.arange(prompt)
    want, absolute = rr.rows(qp, got_k, f(v0[0]), pos[None] <= pos[:, None], pos)
    rr.check(f(out0.read(np.uint16, (prompt, heads, D))), want, absolute, dt, "prompt")

    def check_steps(what):
        cache = [f(b.read(np.uint16, (pool, page, kv, D))) for b in (ck, cv)]
        for s in range(steps):
            got = f(outs[s].read(np.uint16, (requests, heads, D)))
            rq = f(keep[9 * s + 5].read(np.uint16, (requests, heads, D)))
            for r in range(requests):
                n = int(begin[r]) + s + 1
                own = [np.stack([c[table[r, j // page], j % page] for j in range(n)]) for c in cache]
                assert (np.abs(own[0][n - 1] - turn(f(ks[s, r, 0]), prompt + n - 1)) <= rr.HALF[dt] * np.abs(own[0][n - 1]) * 1.01 + 2.0 ** -20).all()
                want, absolute = rr.rows(rq[r][None], np.concatenate((got_k, own[0])), np.concatenate((f(v0[0]), own[1])), np.ones((1, prompt + n), bool),
                                         np.array([prompt + n - 1]))
                rr.check(got[r][None], want, absolute, dt, f"{what}, step {s}, request {r}")

    check_steps("one batch")
    eager = [o.read(np.uint16, (requests, heads, D)) for o in outs]
    g = rr.Captured(queue, all_steps)
    for _ in range(3):
        for o in outs:
            o.write(np.full(requests * heads * D, POISON, np.uint16))
        g.replay()
        for a, o in zip(eager, outs):
            assert np.array_equal(a, o.read(np.uint16, (requests, heads, D)))
    g.close()
    L.zdraw_hip_release_queue(queue)
