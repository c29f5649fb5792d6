"""What of the attention under masks, over a shared prefix and of the cache append can be checked without a GPU: struct sizes,
calls without a queue, how rows are laid on workgroups, the compiled code's hand-kept distances, and the reference itself."""
import ctypes as C
import os
import shutil

import numpy as np
import pytest

from tests import rangeref as rr
from zdraw_amd import build, hip

needs_hipcc = pytest.mark.skipif(not (os.path.exists("/opt/rocm/bin/hipcc") or shutil.which("hipcc")), reason="needs hipcc")


def test_struct_sizes():
    L = hip.lib()
    structs = (hip.MaskedAttn, hip.MaskOperands, hip.SharedAttn, hip.SharedOperands, hip.KvAppend, hip.AppendOperands)
    sizes = (176, 40, 232, 40, 248, 56)
    text = open(os.path.join(build.ROOT, "include", "zdraw_hip.h")).read()
    names = ("MASKED_ATTN", "MASK_OPERANDS", "SHARED_ATTN", "SHARED_OPERANDS", "KV_APPEND", "APPEND_OPERANDS")
    for i, (s, n, name) in enumerate(zip(structs, sizes, names)):
        assert L.zdraw_hip_abi_sizeof(9 + i) == C.sizeof(s) == n
        assert f"#define ZDRAW_HIP_ABI_{name}_SIZE {n}" in text


def test_calls_without_a_queue():
    L = hip.lib()
    for n, fn in ((4, "attention_masked"), (6, "attention_shared"), (6, "kv_append")):
        for suffix in ("", "_enc"):
            assert getattr(L, f"zdraw_hip_run_{fn}{suffix}")(None, *[None] * n, None, None) == hip.ERR_HANDLE
            assert hip.last_error()
    assert L.zdraw_hip_attention_masked_workspace(None, None) == 0 and L.zdraw_hip_attention_shared_workspace(None, None) == 0


def plan(rows, groups, keys, cus=256):
    t, r, s = C.c_uint32(9), C.c_uint32(9), C.c_uint32(9)
    hip.lib().zdraw_hip_masked_plan(rows, groups, keys, cus, C.byref(t), C.byref(r), C.byref(s))
    return t.value, r.value, s.value


def test_layout_of_named_calls():
    assert plan(4, 32, 8191) == (32, 1, 16)          # a token of four sequences, eight key heads: 512 workgroups
    assert plan(4 * 77, 8, 39) == (32, 10, 1)        # a short prompt
    assert plan(4 * 1500, 8, 750) == (128, 47, 1)    # a longer one: 1504 tiles of 32 rows
    assert plan(4 * 128, 8, 16320) == (128, 4, 16)   # 128 rows at the end of a long text
    assert plan(5632, 24, 5632) == (128, 44, 1)
    assert plan(0, 8, 100) == plan(8, 0, 100) == plan(8, 8, 100, 0) == plan(1 << 22, 8, 100) == plan(8, 8, 1 << 24) == (0, 0, 0)


def test_layout_invariants():
    rng = np.random.default_rng(3)
    for _ in range(3000):
        rows, groups, keys = (int(np.exp(rng.uniform(0, np.log(m)))) for m in (400000, 3000, 200000))
        tile, tiles, splits = plan(rows, groups, keys)
        assert tile in (32, 128) and tiles == -(-rows // tile)
        assert 1 <= splits <= 64
        if splits > 1:  # two workgroups a CU at most, and no share under 256 keys
            assert tiles * groups * splits <= 512 and keys // splits >= 256 and keys >= 768


@needs_hipcc
@pytest.mark.parametrize("name", ["attn_masked.hip", "kv_append.hip"])
def test_hand_kept_distances(name):
    # direct-to-LDS loads are assembly statements: nothing but the source may write M0, and none may read a scalar register
    # that a vector instruction has just written
    src = os.path.join(build.CSRC, name)
    bad = build.vmem_sgpr_hazards(src) + build.kernarg_overreads(src) + build.early_store_data_writes(src) + build.early_mfma_result_uses(src)
    bad += build.m0_writes(src, "attn_rows_kernel|attn_keys_kernel")
    assert not bad, "\n".join(bad[:20])


def test_the_reference_against_differences():
    """rows() by its two ways, and against a softmax written out, with a row that sees nothing."""
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((5, 4, 128)), rng.standard_normal((7, 2, 128)), rng.standard_normal((7, 2, 128))
    seen = rng.random((5, 7)) < 0.6
    seen[2] = False
    slopes = np.array([0.5, 0.25, 0.125, 0.0625], np.float32)
    pos = np.arange(5) + 2
    out, absolute = rr.rows(q, k, v, seen, pos, cap=3.0, slopes=slopes)
    assert (out[2] == 0).all() and (np.abs(out) <= absolute + 1e-12).all()
    for h in range(4):
        for i in (0, 1, 3, 4):
            s = 3.0 * np.tanh(k[:, h // 2] @ q[i, h] / np.sqrt(128) / 3.0) - slopes[h] * np.abs(pos[i] - np.arange(7))
            p = np.exp(s) * seen[i]
            assert np.allclose(out[i, h], p @ v[:, h // 2] / p.sum(), atol=1e-12)
    dirty = v.copy()
    dirty[0, 0, 0] = np.inf  # the other way, row by row
    again, _ = rr.rows(q, k, dirty, seen, pos, cap=3.0, slopes=slopes)
    assert np.allclose(again[..., 1:], out[..., 1:], atol=1e-12)
