"""Attention over row ranges and the cache append in 64 bits, the 16-bit types as numpy arrays, and how far a kernel that
rounds as the library says it does may be off."""
import ctypes as C

import numpy as np

from zdraw_amd import hip, host

D = 128
HALF = {hip.BF16: 2.0 ** -8, hip.F16: 2.0 ** -11}  # half a step of the type, relative: eps / 2


def bits(x, dtype):
    """f32 -> the type's bits (nearest even)."""
    x = np.asarray(x, np.float32)
    if dtype == hip.BF16:
        b = host.f32_to_bf16_bits(np.nan_to_num(x, nan=0.0, posinf=np.inf, neginf=-np.inf))
        return np.where(np.isnan(x), np.uint16(0x7FC0), b).astype(np.uint16)
    with np.errstate(over="ignore"):
        return x.astype(np.float16).view(np.uint16)


def value(b, dtype):
    return host.bf16_bits_to_f32(b).astype(np.float64) if dtype == hip.BF16 else np.asarray(b, np.uint16).view(np.float16).astype(np.float64)


def rows(q, k, v, seen, pos, scale=None, cap=0.0, slopes=None, key_pos=None):
    """q [n][heads][D], k, v [keys][kv][D] (f64), seen [n][keys], pos [n]: outputs [n][heads][D] and, per output, the sum of the
    probabilities times |v| (what a relative error of the probabilities is multiplied by)."""
    n, heads, _ = q.shape
    keys, kv, _ = k.shape
    out, absolute = np.zeros(q.shape), np.zeros(q.shape)
    if keys == 0:
        return out, absolute
    scale = 1.0 / np.sqrt(D) if not scale else float(np.float32(scale))
    key_pos = np.arange(keys) if key_pos is None else key_pos
    with np.errstate(all="ignore"):
        for h in range(heads):
            kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
            if all(np.isfinite(x).all() for x in (q[:, h], kh, vh)):  # all rows at once
                s = (q[:, h] @ kh.T) * scale
                if cap:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s - float(slopes[h]) * np.abs(np.asarray(pos)[:, None] - key_pos[None])
                s = np.where(seen, s, -np.inf)
                top = s.max(1, keepdims=True)
                p = np.exp(s - np.where(top == -np.inf, 0.0, top))
                total = p.sum(1, keepdims=True)
                p = p / np.where(total == 0, 1.0, total)
                out[:, h], absolute[:, h] = p @ vh, p @ np.abs(vh)
                continue
            for i in range(n):
                j = np.nonzero(seen[i])[0]
                if len(j) == 0:
                    continue
                s = (kh[j] @ q[i, h]) * scale
                if cap:
                    s = cap * np.tanh(s / cap)
                if slopes is not None:
                    s = s - float(slopes[h]) * np.abs(pos[i] - key_pos[j])
                top = s.max()
                if top == -np.inf:
                    continue
                p = np.exp(s - top)
                p = p / p.sum()
                out[i, h] = (p[:, None] * vh[j]).sum(0)
                absolute[i, h] = (p[:, None] * np.abs(vh[j])).sum(0)
    return out, absolute


def tolerance(want, absolute, dtype, scores=32.0):
    """Half a step of the output's rounding, half a step on every probability as it meets V, and what f32 leaves: scores of
    magnitude `scores` (sum of |q_i k_i| / sqrt(D)) through 128 additions, exponentials and sums, 2^-24 each."""
    f32 = 2.0 ** -24 * (128 * scores + 4096)
    return HALF[dtype] * np.abs(want) + (HALF[dtype] + f32) * absolute * (1 + HALF[dtype]) + 2.0 ** -24


def check(got, want, absolute, dtype, what, scores=32.0):
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(got), nan), f"{what}: NaN where none is, or none where one is: {np.argwhere(np.isnan(got) != nan)[:4].tolist()}"
    inf = np.isinf(want)
    assert np.array_equal(got[inf], want[inf]), f"{what}: infinities"
    ok = ~(nan | inf)
    with np.errstate(invalid="ignore"):
        err = np.abs(got - want)
    bad = ok & ~(err <= tolerance(want, absolute, dtype, scores))
    if bad.any():
        i = tuple(np.argwhere(bad)[0])
        raise AssertionError(f"{what}: {bad.sum()} of {ok.sum()} outputs off, first at {i}: {got[i]} for {want[i]}, allowed {tolerance(want, absolute, dtype, scores)[i]}")


def dense(dst, shape, pad=(0, 0, 0)):
    """Strides of [a][b][c][D] with `pad` extra elements per row, token and segment; the elements that it spans."""
    row = D + pad[0]
    tok = shape[2] * row + pad[1]
    seg = shape[1] * tok + pad[2]
    dst[0], dst[1], dst[2] = seg, tok, row
    return shape[0] * seg


def spread(x, strides, size, fill):
    """x [a][b][c][D] laid out by `strides` in an array of `size` elements, `fill` between them."""
    out = np.full(size, fill, x.dtype)
    a, b, c, _ = x.shape
    at = (np.arange(a)[:, None, None, None] * strides[0] + np.arange(b)[None, :, None, None] * strides[1]
          + np.arange(c)[None, None, :, None] * strides[2] + np.arange(D))
    out[at] = x
    return out


def gather(flat, strides, shape):
    a, b, c, _ = shape
    at = (np.arange(a)[:, None, None, None] * strides[0] + np.arange(b)[None, :, None, None] * strides[1]
          + np.arange(c)[None, None, :, None] * strides[2] + np.arange(D))
    return flat[at]


def stream_of(queue):
    return C.c_void_p((C.c_void_p * 2).from_address(queue)[1])  # a queue is a device and a stream


class Captured:
    """What `enqueue(batch)` puts on a queue, as a graph that can be replayed there."""

    def __init__(self, queue, enqueue):
        L = hip.lib()
        self.queue, self.graph, self.run = queue, C.c_void_p(), C.c_void_p()
        batch = L.zdraw_hip_batch_begin(queue)
        assert L.hipStreamBeginCapture(stream_of(queue), C.c_int(2)) == 0
        rc = enqueue(batch)
        assert L.hipStreamEndCapture(stream_of(queue), C.byref(self.graph)) == 0
        assert rc == 0, hip.last_error()
        assert L.zdraw_hip_batch_end(batch) == 0
        assert L.hipGraphInstantiate(C.byref(self.run), self.graph, None, None, C.c_size_t(0)) == 0

    def nodes(self):
        n = C.c_size_t(0)
        assert hip.lib().hipGraphGetNodes(self.graph, None, C.byref(n)) == 0
        return n.value

    def replay(self):
        L = hip.lib()
        assert L.hipGraphLaunch(self.run, stream_of(self.queue)) == 0
        assert L.hipStreamSynchronize(stream_of(self.queue)) == 0

    def close(self):
        L = hip.lib()
        assert L.hipGraphExecDestroy(self.run) == 0 and L.hipGraphDestroy(self.graph) == 0
