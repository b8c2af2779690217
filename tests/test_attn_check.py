"""What the attention entries refuse, before any device is touched
(katali_hip_attn_check and the argument checks of the calls), the layout of
their descriptors, and how rows and keys are spread over workgroups."""
import ctypes as C
import os
import subprocess
import tempfile

import numpy as np
import pytest

import katali_hip as K

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


class Ptr:
    def __init__(self, p):
        self.ptr = p


def desc(**kw):
    a = dict(kv_type=K.F16, n_head=8, n_kv_head=2, head_dim=128, n_seq=3, kv_len=Ptr(4096), max_kv=100,
             kv_seq_stride=25600, kv_row_stride=256, kv_head_stride=128, scale=0.1)
    a.update(kw)
    d = K.KataliHip.attn_desc(**a)
    return d


@pytest.fixture(scope="module")
def lib():
    return K.KataliHip()


@pytest.mark.parametrize("kw,rc", [
    ({}, 0),
    (dict(kv_type=K.F32), 0), (dict(kv_type=K.BF16), 0), (dict(kv_type=12), K.E_UNSUPPORTED),
    (dict(head_dim=64), 0), (dict(head_dim=96), K.E_UNSUPPORTED), (dict(head_dim=0), K.E_UNSUPPORTED),
    (dict(n_head=7), K.E_INVALID), (dict(n_kv_head=0), K.E_INVALID), (dict(n_head=0), K.E_INVALID),
    (dict(n_head=1026), K.E_INVALID), (dict(n_head=1024, n_kv_head=1), 0),
    (dict(n_seq=0), K.E_INVALID), (dict(n_seq=65536), K.E_INVALID),
    (dict(max_q=0), K.E_INVALID), (dict(max_q=2), K.E_INVALID), (dict(n_rows=4), K.E_INVALID),
    (dict(max_q=2, n_rows=4, q_start=Ptr(64)), 0), (dict(n_rows=0, q_start=Ptr(64)), 0),
    (dict(kv_len=None), K.E_INVALID),
    (dict(max_kv=0), 0), (dict(max_kv=0x7FFFF000), K.E_UNSUPPORTED), (dict(max_kv=0x7FFFEFFF), 0),
    (dict(kv_row_stride=260), K.E_INVALID), (dict(kv_head_stride=4), K.E_INVALID), (dict(kv_seq_stride=1), K.E_INVALID),
    (dict(kv_type=K.F32, kv_row_stride=260), 0), (dict(kv_row_stride=1 << 26), K.E_UNSUPPORTED),
    (dict(kv_seq_stride=1 << 60), K.E_UNSUPPORTED),
    (dict(scale=float("nan")), K.E_INVALID), (dict(scale=float("inf")), K.E_INVALID),
    (dict(softcap=-1.0), K.E_INVALID), (dict(softcap=float("inf")), K.E_INVALID),
    (dict(n_rows=(1 << 22) + 1, max_q=1, n_head=1, n_kv_head=1, q_start=Ptr(64)), K.E_UNSUPPORTED),
    (dict(n_rows=1 << 22, max_q=1, n_head=1, n_kv_head=1, q_start=Ptr(64)), 0),
    (dict(n_seq=65535, n_rows=65535, n_head=512, n_kv_head=1), K.E_UNSUPPORTED),
    (dict(n_seq=65535, n_rows=65535, n_head=128, n_kv_head=1), 0),
    (dict(n_seq=64, n_rows=1 << 16, max_q=1 << 15, q_start=Ptr(64)), K.E_UNSUPPORTED),
    (dict(n_seq=64, n_rows=1 << 16, max_q=1 << 14, q_start=Ptr(64)), 0),
    (dict(n_rows=1 << 28, max_q=1 << 28, q_start=Ptr(64)), K.E_UNSUPPORTED),
    (dict(n_seq=65535, n_rows=1 << 20, max_q=1 << 20, q_start=Ptr(64)), K.E_UNSUPPORTED),
])
def test_descriptor_rules(lib, kw, rc):
    assert lib.lib.katali_hip_attn_check(C.byref(desc(**kw)), None) == rc
    if rc:
        assert lib.lib.katali_hip_last_error()


def test_short_and_missing_descriptors(lib):
    d = desc()
    d.struct_size -= 4
    assert lib.lib.katali_hip_attn_check(C.byref(d), None) == K.E_INVALID
    assert lib.lib.katali_hip_attn_check(None, None) == K.E_INVALID
    assert lib.lib.katali_hip_attn(None, None, None, None, None) == K.E_INVALID
    assert lib.lib.katali_hip_attn_shared(C.byref(desc()), None, None, None, None, None) == K.E_INVALID
    assert lib.lib.katali_hip_kv_append(C.byref(desc()), None, None, None, None, None, None, None) == K.E_INVALID


@pytest.mark.parametrize("kw,rc", [
    ({}, 0), (dict(n_prefix=0), K.E_INVALID), (dict(k=Ptr(None)), K.E_INVALID), (dict(v=Ptr(None)), K.E_INVALID),
    (dict(k=Ptr(8)), K.E_INVALID), (dict(row_stride=100), K.E_INVALID), (dict(head_stride=3), K.E_INVALID),
    (dict(n_prefix=0x7FFFF000 - 100), K.E_UNSUPPORTED), (dict(n_prefix=0x7FFFF000 - 101), 0),
])
def test_prefix_rules(lib, kw, rc):
    a = dict(n_prefix=50, k=Ptr(4096), v=Ptr(8192), row_stride=256, head_stride=128)
    a.update(kw)
    p = K.KataliHip.attn_prefix(**a)
    assert lib.lib.katali_hip_attn_check(C.byref(desc()), C.byref(p)) == rc


@pytest.mark.parametrize("q,k,v,out", [(None, 16, 16, 1 << 20), (16, None, 16, 1 << 20), (16, 16, None, 1 << 20),
                                        (16, 16, 16, None), (8, 16, 16, 1 << 20), (16, 24, 16, 1 << 20),
                                        (16, 16, 20, 1 << 20), (16, 16, 16, (1 << 20) + 4), (16, 1 << 20, 1 << 20, 16),
                                        (16, 1 << 20, 1 << 20, 16 + 3 * 8 * 128 * 4 - 16)])
def test_buffers_of_attn(lib, q, k, v, out):
    assert lib.lib.katali_hip_attn(C.byref(desc()), q, k, v, out) == K.E_INVALID


@pytest.mark.parametrize("kw", [dict(n_rot=3), dict(n_rot=130), dict(base=0.0), dict(base=-1.0), dict(base=float("nan")),
                                dict(base=float("inf")), dict(eps=-1.0), dict(eps=float("nan"))])
def test_rope_rules(lib, kw):
    a = dict(n_rot=128, base=1e4)
    a.update(kw)
    r = K.KataliHip.rope(**a)
    assert lib.lib.katali_hip_kv_append(C.byref(desc()), C.byref(r), 1 << 12, 1 << 20, 1 << 21, 1 << 22, 1 << 23,
                                        1 << 24) == K.E_INVALID


@pytest.mark.parametrize("i", range(6))
def test_buffers_of_append(lib, i):
    r = K.KataliHip.rope(128, 1e4)
    good = [1 << 14, 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24]
    for bad in (None, good[i] + 8):
        b = list(good)
        b[i] = bad
        assert lib.lib.katali_hip_kv_append(C.byref(desc()), C.byref(r), *b) == K.E_INVALID
    over = list(good)
    over[3] = good[0] + 64   # q_out overlaps q without being it
    assert lib.lib.katali_hip_kv_append(C.byref(desc()), C.byref(r), *over) == K.E_INVALID


def test_layouts():
    src = """
#include <stdio.h>
#include <stddef.h>
#include "katali_hip.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu %zu %zu\\n", sizeof(KataliHipAttn), offsetof(KataliHipAttn, q_start),
         offsetof(KataliHipAttn, scale), offsetof(KataliHipAttn, doc_end), sizeof(KataliHipAttnPrefix),
         offsetof(KataliHipAttnPrefix, head_stride), sizeof(KataliHipRope), offsetof(KataliHipRope, k_norm_w));
  return 0;
}
"""
    with tempfile.TemporaryDirectory() as d:
        open(os.path.join(d, "t.c"), "w").write(src)
        subprocess.run(["gcc", "-I" + os.path.join(REPO, "include"), os.path.join(d, "t.c"), "-o", os.path.join(d, "t")],
                       check=True)
        vals = [int(x) for x in subprocess.run([os.path.join(d, "t")], capture_output=True, text=True).stdout.split()]
    A, P, R = K.KataliHipAttn, K.KataliHipAttnPrefix, K.KataliHipRope
    assert vals == [C.sizeof(A), A.q_start.offset, A.scale.offset, A.doc_end.offset, C.sizeof(P), P.head_stride.offset,
                    C.sizeof(R), R.k_norm_w.offset]


def test_oracle_bf16_rounds_to_nearest_even():
    import attn_oracle as O
    x = np.asarray([1.0, 1.00390625, 1.01171875, -1.0040, 3.0e38, 1e-40], np.float32)
    raw, val = O.to_cache(x, K.BF16)
    assert val[0] == 1.0 and val[1] == 1.0 and val[2] == 1.015625 and val[3] == -1.0078125
    half = np.abs(val[:4] - x[:4]) <= 2.0 ** -8 * np.abs(x[:4])
    assert half.all() and raw.dtype == np.uint16


@pytest.mark.parametrize("kw", [dict(), dict(softcap=20.0), dict(alibi=True), dict(n_shared=13), dict(causal=False)])
def test_the_two_forms_of_the_oracle_agree(kw):
    import attn_oracle as O
    rng = np.random.default_rng(3)
    c = O.make(rng, 3, [5, 0, 9], [7, 4, 30], 30, 4, 2, 64, K.F16, prefix=[0, 3, 25], lead=1,
               docs=lambda c: (rng.integers(0, 12, c["n_rows"]), rng.integers(0, 40, c["n_rows"])), **kw)
    a, b = O.attn(c), O.attn_wide(c)
    assert np.array_equal(np.isnan(a), np.isnan(b)) and np.nanmax(np.abs(a - b)) < 1e-12
