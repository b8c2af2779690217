"""GPU parity: attention over caches (katali_hip_attn), over a shared prefix
(katali_hip_attn_shared) and the step that stores new rows
(katali_hip_kv_append), through the C ABI, against their definitions in 64
bits. The tolerance is derived in attn_oracle.tolerance."""
import numpy as np
import pytest

import attn_oracle as O
import katali_hip as K

pytestmark = pytest.mark.gpu

TYPES = [K.F32, K.F16, K.BF16]
NAMES = {K.F32: "f32", K.F16: "f16", K.BF16: "bf16"}


def check(hip, c, **kw):
    print(f"[attn] {NAMES[c['t']]} seqs={c['n_seq']} rows={c['nq'].tolist()[:8]} keys={c['kv_len'].tolist()[:8]} "
          f"heads={c['n_head']}/{c['n_kv']}x{c['D']} shared={c['n_shared']}", flush=True)
    got = O.run(hip, c, **kw)
    O.compare(c, got, O.attn(c))
    return got


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_keys", [1, 2, 15, 16, 17, 31, 32, 33, 127, 300, 1025])
def test_one_token(hip, t, D, n_keys):
    rng = np.random.default_rng(n_keys + D)
    c = O.make(rng, 1, [1], [n_keys], n_keys + 5, 8, 2, D, t)
    c["no_start"] = True
    check(hip, c)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n_head,n_kv", [(1, 1), (3, 1), (8, 8), (16, 1), (17, 1), (40, 2), (6, 2)])
def test_head_layouts(hip, t, n_head, n_kv):
    rng = np.random.default_rng(n_head)
    check(hip, O.make(rng, 2, [1, 3], [70, 41], 80, n_head, n_kv, 64, t))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("rows,keys", [(2, 2), (5, 200), (33, 33), (64, 64), (65, 130), (129, 129), (200, 517)])
def test_prompts(hip, t, D, rows, keys):
    rng = np.random.default_rng(rows + D)
    check(hip, O.make(rng, 1, [rows], [keys], keys, 4, 2, D, t))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("softcap,alibi", [(30.0, False), (0.0, True), (50.0, True)])
@pytest.mark.parametrize("rows,keys", [(1, 300), (70, 140)])
def test_cap_and_bias(hip, t, softcap, alibi, rows, keys):
    rng = np.random.default_rng(rows)
    check(hip, O.make(rng, 2, [rows, max(1, rows // 3)], [keys, keys - 9], keys, 4, 2, 128, t, softcap=softcap,
                      alibi=alibi, std=4.0 if softcap else 1.3))


def documents(c):
    """Documents of odd lengths; some rows see nothing: an empty one, one past
    the row's end, and bounds far outside."""
    rng = np.random.default_rng(5)
    a, b = np.zeros(c["n_rows"], np.int64), np.full(c["n_rows"], 2 ** 31 - 1)
    for s in range(c["n_seq"]):
        n = int(c["kv_len"][s]) + c["n_shared"]
        cuts = np.concatenate([[0], np.sort(rng.integers(0, n + 1, 4)), [n]])
        for i in range(int(c["nq"][s])):
            pos = n - int(c["nq"][s]) + i
            w = np.searchsorted(cuts, pos, side="right")
            row = int(c["q_start"][s]) + i
            a[row], b[row] = cuts[w - 1], cuts[min(w, len(cuts) - 1)]
            if i % 7 == 3:
                a[row], b[row] = [(5, 5), (2 ** 31 - 1, 0), (-2 ** 31, -2 ** 31), (pos + 1, 2 ** 31 - 1)][i % 4]
    return a, b


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("rows,keys", [([1, 1, 1], [40, 7, 333]), ([90, 3, 64], [90, 200, 65])])
def test_documents(hip, t, causal, rows, keys):
    rng = np.random.default_rng(1)
    check(hip, O.make(rng, 3, rows, keys, max(keys), 4, 2, 64, t, causal=causal, docs=documents))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,shared", [(1, 0), (1, 900), (50, 0)])
def test_bias_of_rows_that_see_far_keys_only(hip, t, rows, shared):
    """Rows whose documents end far before them: biases of several hundred,
    the same for all their keys but for a few units, cost no bits."""
    rng = np.random.default_rng(21)

    def far(c):
        return np.zeros(c["n_rows"], int), np.asarray([40 + 3 * (i % 9) for i in range(c["n_rows"])])
    check(hip, O.make(rng, 3, [rows] * 3, [1000, 800, 900], 1000, 8, 2, 128, t, alibi=True, docs=far, n_shared=shared))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("prefix", [[0, 30, 2 ** 31 - 1], [-5, 61, 100]])
def test_prefix_seen_from_both_sides(hip, t, prefix):
    rng = np.random.default_rng(2)
    check(hip, O.make(rng, 3, [60, 70, 99], [60, 75, 99], 99, 2, 1, 128, t, prefix=prefix, alibi=True))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_ragged_rows(hip, t):
    """Sequences without rows, without keys, with fewer keys than rows, and
    packed rows before, behind and past max_q that are left as they were."""
    rng = np.random.default_rng(3)
    c = O.make(rng, 5, [0, 4, 1, 9, 2], [10, 0, 5, 3, 40], 40, 4, 1, 64, t, lead=3, tail=5)
    check(hip, c)
    c = O.make(rng, 2, [5, 2], [30, 20], 40, 4, 1, 64, t, max_q=3)
    want = O.attn(c)
    want[3:5] = np.nan   # rows past max_q of sequence 0
    O.compare(c, O.run(hip, c), want)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows", [1, 50])
@pytest.mark.parametrize("shared", [0, 70])
def test_no_own_keys(hip, t, rows, shared):
    """Caches of no rows: zeros, or the shared keys alone."""
    rng = np.random.default_rng(22)
    c = O.make(rng, 3, [rows] * 3, [0, 0, 0], 0, 4, 2, 64, t, n_shared=shared, causal=False)
    check(hip, c)
    check(hip, {**c, "causal": True})


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_not_causal(hip, t):
    rng = np.random.default_rng(4)
    check(hip, O.make(rng, 2, [37, 50], [100, 50], 100, 4, 2, 128, t, causal=False, alibi=True))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_head_major_cache(hip, t):
    """A cache laid out [key head][sequence][row + 3 spare][D]."""
    rng = np.random.default_rng(6)
    c = O.make(rng, 2, [1, 20], [50, 45], 50, 6, 3, 64, t)
    rows = 53

    def lay(x):
        y = np.zeros((3, 2, rows, 64), x.dtype)
        y[:, :, :50] = x.transpose(2, 0, 1, 3)
        return hip.to_device(y)
    got = O.run(hip, c, k=lay(c["k_raw"]), v=lay(c["v_raw"]), strides=(rows * 64, 64, 2 * rows * 64))
    O.compare(c, got, O.attn(c))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("rows,keys", [(1, 100), (40, 100), (100, 100)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_values_nobody_sees(hip, t, rows, keys, bad):
    """NaN and infinities in keys and values behind a sequence's end, and in
    rows that only later queries see."""
    rng = np.random.default_rng(7)
    c = O.make(rng, 2, [rows, rows], [keys, keys - 30 if rows < 80 else keys], keys + 20, 4, 2, 128, t)
    for n in ("k", "v"):
        for s in range(2):
            at = int(c["kv_len"][s])
            c[n][s, at:] = bad
            if rows > 1:
                c[n][s, at - 2] = bad
        raw, _ = O.to_cache(c[n], t)
        c[n + "_raw"] = raw
    want = O.attn({**c, "k": np.nan_to_num(c["k"], posinf=0, neginf=0), "v": np.nan_to_num(c["v"], posinf=0, neginf=0)})
    if rows > 1:   # the last two rows of each sequence see the bad key
        for s in range(2):
            want[int(c["q_start"][s + 1]) - 2:int(c["q_start"][s + 1])] = np.nan
    got = O.run(hip, c)
    seen = np.isnan(want).all(axis=(1, 2))
    assert not np.isfinite(got[seen]).any() or rows == 1
    got[seen] = 777.0
    O.compare(c, got, want)


@pytest.mark.parametrize("t", [K.F16, K.BF16], ids=NAMES.get)
@pytest.mark.parametrize("size", [1e-6, 1e6])
def test_size_of_q(hip, t, size):
    """q far from one, the scale bringing scores back."""
    rng = np.random.default_rng(8)
    c = O.make(rng, 1, [40], [90], 90, 2, 1, 128, t)
    want = O.attn(c)
    c["q"] = (c["q"].astype(np.float64) * size).astype(np.float32)
    c["scale"] = c["scale"] / size
    got = O.run(hip, c)
    c["q"] = (c["q"] / np.float32(size))
    O.compare(c, got, want)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n_seq,rows,own,shared", [(2, 1, 1, 17), (5, 1, 33, 500), (9, 3, 20, 129), (3, 50, 60, 90),
                                                    (1, 1, 30, 40)])
def test_shared(hip, t, D, n_seq, rows, own, shared):
    rng = np.random.default_rng(n_seq)
    nq = [rows] + [int(rng.integers(1, rows + 1)) for _ in range(n_seq - 1)]
    nk = [own] + [int(rng.integers(q, own + 1)) for q in nq[1:]]
    check(hip, O.make(rng, n_seq, nq, nk, own, 8, 2, D, t, n_shared=shared, alibi=True))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("how", ["bare", "cap", "bias"])
@pytest.mark.parametrize("n_seq,rows,shared", [(3, 1, 32), (9, 3, 32), (9, 3, 33), (20, 1, 700), (40, 2, 64), (2, 8, 300)])
def test_shared_few_and_many_rows(hip, t, D, how, n_seq, rows, shared):
    """Rows of all sequences together from a few (12) to several tiles, one
    stage of shared keys and many."""
    rng = np.random.default_rng(n_seq + shared)
    check(hip, O.make(rng, n_seq, [rows] * n_seq, [20] * n_seq, 20, 8, 2, D, t, n_shared=shared, alibi=how == "bias",
                      softcap=20.0 if how == "cap" else 0.0))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
def test_shared_masks(hip, t):
    """Documents and prefixes that end inside the shared keys, sequences
    without rows or own keys, a cap."""
    rng = np.random.default_rng(11)
    check(hip, O.make(rng, 4, [2, 0, 1, 2], [30, 5, 1, 2], 30, 6, 2, 64, t, n_shared=111, docs=documents))
    check(hip, O.make(rng, 4, [2, 0, 1, 2], [30, 5, 1, 2], 30, 6, 2, 64, t, n_shared=111, softcap=20.0, std=4.0,
                      prefix=[0, 50, 120, 200], lead=2, tail=1))


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("how", ["bare", "masks", "unseen"])
def test_parts_of_keys(hip, t, D, how):
    """Keys in parts whose results are joined: sequences that fill all parts, some,
    one and none, rows that see keys of one part only, one row and several tiles of rows."""
    rng = np.random.default_rng(D)
    masks = dict(docs=documents, alibi=True, softcap=30.0, std=3.0, prefix=[0, 1500, 9, 3]) if how == "masks" else {}
    for rows, n_head in ((1, 8), (9, 14)):
        c = O.make(rng, 4, [rows, rows, 1, 0], [1900, 1300, 33, 0], 1900, n_head, 2, D, t, **masks)
        want = O.attn(c)
        if how == "unseen":   # keys behind each sequence's end
            for s in range(4):
                for name in ("k", "v"):
                    c[name][s, c["kv_len"][s]:] = np.inf
            for name in ("k", "v"):
                c[name + "_raw"] = O.to_cache(c[name], t)[0]
        print(f"[attn] parts {NAMES[t]} {how} rows={rows} of {D}", flush=True)
        O.compare(c, O.run(hip, c), want)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("how", ["bare", "cap", "masks"])
@pytest.mark.parametrize("n_seq,rows,shared", [(2, 1, 777), (3, 1, 1001), (9, 3, 790), (21, 2, 1600)])
def test_long_shared_prefix(hip, t, D, how, n_seq, rows, shared):
    """Shared keys enough that the rows of all sequences walk them together:
    one tile of rows to several, own keys from none to many."""
    rng = np.random.default_rng(n_seq + shared)
    nk = [300] + [int(rng.integers(rows, 300)) for _ in range(n_seq - 1)]
    nk[-1] = 0
    nq = [rows] * (n_seq - 1) + [0]
    masks = dict(docs=documents, alibi=True, prefix=[900] * n_seq) if how == "masks" else {}
    check(hip, O.make(rng, n_seq, nq, nk, 300, 8, 2, D, t, n_shared=shared, softcap=20.0 if how == "cap" else 0.0, **masks))


# rows x keys from which tiles of 64 rows and more are taken (attn_plan), by
# head width: 8 key heads of 4 query heads, one sequence, 256 CUs
WIDE = {64: 900, 128: 640, 256: 460}


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("how", ["bare", "masks", "prefix", "unseen"])
def test_wide_tiles(hip, t, D, how):
    rng = np.random.default_rng(D)
    n = WIDE[D] + 3
    if how == "bare":
        c = O.make(rng, 2, [n, n // 3], [n + 17, n // 2], n + 17, 32, 8, D, t, lead=1, tail=2)
    elif how == "masks":
        c = O.make(rng, 2, [n, n // 2], [n, n], n, 32, 8, D, t, docs=documents, alibi=True, softcap=30.0, std=3.0)
    elif how == "prefix":   # a shared prefix walked ahead of own keys, seen from both sides beyond its end
        c = O.make(rng, 2, [n, 5], [n, 70], n, 32, 8, D, t, n_shared=77, prefix=[150, 90], alibi=True)
    else:                   # the last rows' key and what lies behind the end
        c = O.make(rng, 1, [n], [n], n + 9, 32, 8, D, t)
        for name in ("k", "v"):
            c[name][0, n - 2:] = np.nan
            c[name + "_raw"] = O.to_cache(c[name], t)[0]
    print(f"[attn] wide {NAMES[t]} {how} rows={c['nq'].tolist()} keys={c['kv_len'].tolist()} of {D}", flush=True)
    fine = {**c, "k": np.nan_to_num(c["k"]), "v": np.nan_to_num(c["v"])}
    want, got = O.attn_wide(fine), O.run(hip, c)
    if how == "unseen":
        assert np.isnan(got[n - 2:]).all()
        got[n - 2:], want[n - 2:] = 777.0, np.nan
    O.compare(c, got, want)


def test_long_cache_passes_32_bits(hip):
    """Keys whose byte offsets pass 2^32: a cache of 2.5 million rows spread
    over 5 GB, of which the last rows are read (a document's start)."""
    H, KV, D, n, stride = 2, 1, 64, 40_000_000 // 16, 1024
    rng = np.random.default_rng(12)
    tail = 70
    k, kv = O.to_cache(rng.standard_normal((tail, D)), K.F16)
    v, vv = O.to_cache(rng.standard_normal((tail, D)), K.F16)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    kd, vd = hip.alloc(n * stride * 2), hip.alloc(n * stride * 2)
    for i in range(tail):
        at = (n - tail + i) * stride * 2
        for d, src in ((kd, k), (vd, v)):
            row = np.ascontiguousarray(src[i])
            hip.check(hip.lib.katali_hip_upload(d.ptr + at, row.ctypes.data, row.nbytes))
    out = hip.alloc(H * D * 4)
    i32 = lambda x: hip.to_device(np.asarray([x], np.int32))  # noqa: E731
    d = hip.attn_desc(K.F16, H, KV, D, n_seq=1, kv_len=i32(n), max_kv=n, kv_seq_stride=n * stride,
                      kv_row_stride=stride, kv_head_stride=D, scale=0.125, doc_start=i32(n - tail))
    hip.attn(d, hip.to_device(q), kd, vd, out)
    got = out.download(np.float32).reshape(H, D)
    for h in range(H):
        x = 0.125 * (kv @ q[0, h].astype(np.float64))
        p = np.exp(x - x.max())
        want = (p / p.sum()) @ vv
        assert np.linalg.norm(got[h] - want) <= 2e-5 * np.linalg.norm(want)


def append_case(rng, t, D, nq, kv_len, max_kv, n_head=6, n_kv=2, **kw):
    c = O.make(rng, len(nq), nq, kv_len, max_kv, n_head, n_kv, D, t, **kw)
    n = c["n_rows"]
    return c, rng.standard_normal((n, n_kv, D)).astype(np.float32) * 2, rng.standard_normal((n, n_kv, D)).astype(np.float32)


@pytest.mark.parametrize("t", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("D,n_rot,interleaved", [(64, 64, False), (128, 64, True), (128, 128, False), (256, 64, False),
                                                 (256, 256, True), (128, 0, False), (64, 2, False), (128, 34, True)])
@pytest.mark.parametrize("norm", [True, False])
def test_append(hip, t, D, n_rot, interleaved, norm):
    print(f"[append] {NAMES[t]} D={D} n_rot={n_rot} interleaved={interleaved} norm={norm}", flush=True)
    rng = np.random.default_rng(D + n_rot)
    # a sequence without rows, one whose rows' positions pass its cache, one with fewer keys than rows
    c, kn, vn = append_case(rng, t, D, [1, 0, 7, 3], [9, 4, 30, 2], 30, lead=1, tail=2)
    pos0, base, eps = 70001, 1e6, 1e-6
    qw, kw = [(1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2)] if norm else (None, None)
    i32 = lambda a: hip.to_device(np.asarray(a, np.int32))  # noqa: E731
    d = hip.attn_desc(t, 6, 2, D, n_seq=4, n_rows=c["n_rows"], max_q=7, max_kv=30, q_start=i32(c["q_start"]),
                      kv_len=i32(c["kv_len"]), kv_seq_stride=30 * 2 * D, kv_row_stride=2 * D, kv_head_stride=D,
                      scale=1.0)
    r = hip.rope(n_rot, base, interleaved=interleaved, pos0=pos0, eps=eps,
                 q_norm_w=None if qw is None else hip.to_device(qw), k_norm_w=None if kw is None else hip.to_device(kw))
    want_q, want_k, want_v, stored = O.append(c, kn, vn, n_rot, base, interleaved, pos0, eps, qw, kw)
    for in_place in (False, True):
        q, k, v = hip.to_device(c["q"]), hip.to_device(c["k_raw"]), hip.to_device(c["v_raw"])
        qo = q if in_place else hip.to_device(np.full(c["q"].shape, 777.0, np.float32))
        hip.kv_append(d, r, q, hip.to_device(kn), hip.to_device(vn), qo, k, v)
        got = qo.download(np.float32).reshape(c["q"].shape)
        none = np.isnan(want_q)
        assert np.array_equal(got[none], c["q"][none] if in_place else np.full(none.sum(), 777.0, np.float32))
        # angles to 2^-24 of a turn in cos and sin, norm and products a few 2^-24
        bar = 16 * 2.0 ** -24
        assert np.abs(got - want_q)[~none].max() <= bar * np.abs(want_q[~none]).max()
        # one rounding to the cache's type on top: half a step of the value
        half = {K.F32: 2.0 ** -24, K.F16: 2.0 ** -11, K.BF16: 2.0 ** -8}[t]
        for buf, raw, want in ((k, c["k_raw"], want_k), (v, c["v_raw"], want_v)):
            g = buf.download(raw.dtype).reshape(raw.shape)
            assert np.array_equal(g[~stored], raw[~stored]), "cache rows of other positions were written"
            vals = (g.astype(np.uint32) << 16).view(np.float32) if t == K.BF16 else g
            err = np.abs(vals.astype(np.float64) - want)[stored]
            assert (err <= half * np.abs(want[stored]) + bar * np.abs(want[stored]).max()).all()
        g = v.download(c["v_raw"].dtype).reshape(c["v_raw"].shape)
        for s in range(4):   # v goes in with one rounding and nothing else
            for i in range(int(c["nq"][s])):
                p = int(c["kv_len"][s]) - int(c["nq"][s]) + i
                if 0 <= p < 30:
                    assert np.array_equal(g[s, p], O.to_cache(vn[int(c["q_start"][s]) + i], t)[0])


@pytest.mark.parametrize("pos", [0, 1, 131071, 10_000_000, 2 ** 31 - 5000])
def test_append_far_positions(hip, pos):
    rng = np.random.default_rng(13)
    c, kn, vn = append_case(rng, K.F32, 128, [2], [2], 2)
    i32 = lambda a: hip.to_device(np.asarray(a, np.int32))  # noqa: E731
    d = hip.attn_desc(K.F32, 6, 2, 128, n_seq=1, n_rows=2, max_q=2, max_kv=2, q_start=i32([0, 2]), kv_len=i32([2]),
                      kv_seq_stride=512, kv_row_stride=256, kv_head_stride=128, scale=1.0)
    want_q, want_k, _, _ = O.append(c, kn, vn, 128, 1e4, False, pos, 0.0, None, None)
    k, v, qo = hip.to_device(c["k_raw"]), hip.to_device(c["v_raw"]), hip.alloc(c["q"].nbytes)
    hip.kv_append(d, hip.rope(128, 1e4, pos0=pos), hip.to_device(c["q"]), hip.to_device(kn), hip.to_device(vn), qo, k, v)
    got = qo.download(np.float32).reshape(c["q"].shape)
    # pos * freq in 64 bits, a few 2^-53 of it, in radians: 2^31 * 2^-51 at most
    bar = 16 * 2.0 ** -24 + 2.0 ** -20
    assert np.abs(got - want_q).max() <= bar * np.abs(want_q).max()
    assert np.abs(k.download(np.float32).reshape(want_k.shape) - want_k).max() <= bar * np.abs(want_k).max()


def test_first_call_inside_a_capture_is_refused_or_ready(hip):
    """Scratch is there after the first call: a captured call replays with new
    lengths, between eager calls of other shapes, each equal to its eager run."""
    rng = np.random.default_rng(14)
    c = O.make(rng, 3, [1, 1, 1], [50, 700, 9], 800, 8, 2, 128, K.F16)
    keep = []
    first = O.run(hip, c, keep_out=keep)
    d, q, k, v, o = keep
    hip.graph_begin()
    hip.attn(d, q, k, v, o)
    g = hip.graph_end()
    try:
        kv_len = d._keep[1]
        for lens in ([50, 700, 9], [51, 701, 10], [800, 1, 0], [3, 3, 3]):
            kv_len.upload(np.asarray(lens, np.int32))
            hip.memset(o, 0, o.nbytes)
            hip.graph_launch(g)
            other = O.make(rng, 2, [1, 1], [300, 40], 300, 4, 4, 64, K.BF16)
            O.compare(other, O.run(hip, other), O.attn(other))
            c["kv_len"] = np.asarray(lens)
            got = o.download(np.float32).reshape(3, 8, 128)
            O.compare(c, got, O.attn(c))
            hip.attn(d, q, k, v, o)
            assert np.array_equal(o.download(np.float32).reshape(3, 8, 128), got)
        assert np.isfinite(first).all()
    finally:
        hip.graph_destroy(g)


def test_same_bits_each_time(hip):
    rng = np.random.default_rng(15)
    c = O.make(rng, 4, [1, 1, 1, 1], [900, 20, 1500, 77], 1500, 8, 2, 128, K.BF16, n_shared=700)
    a = O.run(hip, c)
    for _ in range(3):
        assert np.array_equal(O.run(hip, c), a)


def test_steps_of_a_chain(hip):
    """append and attention as a decode loop runs them: a prompt, then single
    tokens into the same caches, against the definition at every step."""
    rng = np.random.default_rng(16)
    H, KV, D, cap, t = 8, 2, 128, 40, K.F16
    k, v = np.zeros((2, cap, KV, D)), np.zeros((2, cap, KV, D))
    kd, vd = hip.to_device(np.zeros((2, cap, KV, D), np.float16)), hip.to_device(np.zeros((2, cap, KV, D), np.float16))
    have = np.zeros(2, np.int64)
    i32 = lambda a: hip.to_device(np.asarray(a, np.int32))  # noqa: E731
    for nq in ([9, 21], [1, 1], [1, 1], [4, 1]):
        nq = np.asarray(nq)
        have = have + nq
        n = int(nq.sum())
        c = O.make(rng, 2, nq, have, cap, H, KV, D, t)
        kn, vn = (rng.standard_normal((n, KV, D)).astype(np.float32) for _ in range(2))
        c["k"], c["v"] = k, v
        want_q, k, v, _ = O.append(c, kn, vn, D, 1e4, False, 0, 1e-6, None, None)
        k, v = k.astype(np.float16).astype(np.float64), v.astype(np.float16).astype(np.float64)
        d = hip.attn_desc(t, H, KV, D, n_seq=2, n_rows=n, max_q=int(nq.max()), max_kv=cap, q_start=i32(c["q_start"]),
                          kv_len=i32(have), kv_seq_stride=cap * KV * D, kv_row_stride=KV * D, kv_head_stride=D,
                          scale=c["scale"])
        q, o = hip.to_device(c["q"]), hip.alloc(c["q"].nbytes)
        hip.kv_append(d, hip.rope(D, 1e4), q, hip.to_device(kn), hip.to_device(vn), q, kd, vd)
        hip.attn(d, q, kd, vd, o)
        # the caches as the device rounded them: a value next to a rounding border may differ by a step
        c["k"] = kd.download(np.float16).reshape(k.shape).astype(np.float64)
        c["v"] = vd.download(np.float16).reshape(v.shape).astype(np.float64)
        assert np.abs(c["k"] - k).max() <= 2.0 ** -10 * np.abs(k).max()
        c["q"] = q.download(np.float32).reshape(c["q"].shape)
        assert np.abs(c["q"] - want_q).max() <= 2.0 ** -19 * np.abs(want_q).max()
        O.compare(c, o.download(np.float32).reshape(c["q"].shape), O.attn(c))
        k, v = c["k"], c["v"]


def test_another_stream(hip):
    """The calls run on the stream that set_stream names, in order with its other work."""
    import ctypes as C
    with open("/proc/self/maps") as f:   # the HIP runtime that the library loaded
        runtime = C.CDLL(next(line.split()[-1] for line in f if "libamdhip64" in line))
    rng = np.random.default_rng(17)
    c = O.make(rng, 3, [1, 1, 1], [400, 30, 1], 400, 8, 2, 128, K.F16)
    want, keep = O.attn(c), []
    O.run(hip, c, keep_out=keep)
    d, q, k, v, o = keep
    s = C.c_void_p()
    assert runtime.hipStreamCreateWithFlags(C.byref(s), 1) == 0
    hip.check(hip.lib.katali_hip_set_stream(s))
    try:
        for _ in range(3):
            hip.memset(o, 0, o.nbytes)
            hip.attn(d, q, k, v, o)
        O.compare(c, o.download(np.float32).reshape(3, 8, 128), want)
    finally:
        hip.check(hip.lib.katali_hip_set_stream(None))
        assert runtime.hipStreamDestroy(s) == 0


def test_first_call_inside_a_capture():
    """In a fresh process: the first attention call allocates the scratch, so
    inside a capture it is refused; after one eager call it may be captured."""
    import os
    import subprocess
    import sys
    here = os.path.dirname(os.path.abspath(__file__))
    code = (
        "import numpy as np, sys\n"
        "import attn_oracle as O, katali_hip as K\n"
        "hip = K.KataliHip(); assert hip.probe()\n"
        "c = O.make(np.random.default_rng(0), 1, [1], [300], 300, 4, 1, 64, K.F32)\n"
        "i32 = lambda a: hip.to_device(np.asarray(a, np.int32))\n"
        "d = hip.attn_desc(K.F32, 4, 1, 64, n_seq=1, kv_len=i32([300]), max_kv=300, kv_seq_stride=19200,\n"
        "                  kv_row_stride=64, kv_head_stride=64, scale=c['scale'])\n"
        "q, k, v, o = hip.to_device(c['q']), hip.to_device(c['k_raw']), hip.to_device(c['v_raw']), hip.alloc(1024)\n"
        "hip.graph_begin()\n"
        "try:\n"
        "    hip.attn(d, q, k, v, o); sys.exit('not refused')\n"
        "except K.HipError as e:\n"
        "    assert e.rc == K.E_INVALID and 'capture' in str(e), e\n"
        "try:\n"
        "    hip.graph_destroy(hip.graph_end())\n"
        "except K.HipError:\n"
        "    pass\n"
        "hip.attn(d, q, k, v, o)\n"
        "hip.graph_begin(); hip.attn(d, q, k, v, o); g = hip.graph_end()\n"
        "for _ in range(3):\n"
        "    hip.memset(o, 0, 1024); hip.graph_launch(g)\n"
        "    got = o.download(np.float32).reshape(1, 4, 64)\n"
        "    O.compare(c, got, O.attn(c))\n"
        "hip.graph_destroy(g); print('fine')\n")
    p = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=100,
                       env={**os.environ, "PYTHONPATH": os.pathsep.join([here, os.path.join(here, "..", "katali-lab_amd")])})
    assert p.returncode == 0 and "fine" in p.stdout, p.stdout + p.stderr
