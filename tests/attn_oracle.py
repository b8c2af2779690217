"""Attention over caches and the step that stores new rows, in 64 bits from
their definitions (include/katali_hip.h), one row and head after another, and
small random calls of them."""
import numpy as np

import katali_hip as K

NP = {K.F32: np.float32, K.F16: np.float16}


def to_cache(x, t):
    """fp32 values as a cache of type t holds them: (raw array, the values)."""
    x = np.ascontiguousarray(x, np.float32)
    if t == K.BF16:
        u = x.view(np.uint32).astype(np.uint64)
        r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)   # nearest even
        r = np.where(np.isnan(x), np.uint16(0x7FC0), r)
        return r, (r.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    r = x.astype(NP[t])
    return r, r.astype(np.float64)


def row_range(c, s, t, row):
    """Position and visible keys [lo, hi) of row t of sequence s."""
    sh = c["n_shared"]
    pos = sh + int(c["kv_len"][s]) - int(c["nq"][s]) + t
    lo, hi = 0, sh + int(c["kv_len"][s])
    if c["causal"]:
        hi = min(hi, max(pos + 1, int(c["prefix_len"][s]) if c["prefix_len"] is not None else pos + 1))
    if c["doc_start"] is not None:
        lo = max(lo, int(c["doc_start"][row]))
    if c["doc_end"] is not None:
        hi = min(hi, int(c["doc_end"][row]))
    return pos, lo, hi


def attn(c):
    """out [n_rows][n_head][D]; NaN where no row is served (left as it was)."""
    H, KV, D = c["n_head"], c["n_kv"], c["D"]
    out = np.full((c["n_rows"], H, D), np.nan)
    for s in range(c["n_seq"]):
        for t in range(int(c["nq"][s])):
            row = int(c["q_start"][s]) + t
            pos, lo, hi = row_range(c, s, t, row)
            for h in range(H):
                g = h // (H // KV)
                k, v = c["k"][s, :int(c["kv_len"][s]), g], c["v"][s, :int(c["kv_len"][s]), g]
                if c["n_shared"]:
                    k, v = np.concatenate([c["pk"][:, g], k]), np.concatenate([c["pv"][:, g], v])
                if lo >= hi:
                    out[row, h] = 0
                    continue
                x = c["scale"] * (k[lo:hi] @ c["q"][row, h].astype(np.float64))
                if c["softcap"]:
                    x = c["softcap"] * np.tanh(x / c["softcap"])
                if c["slopes"] is not None:
                    x = x - float(c["slopes"][h]) * np.abs(pos - np.arange(lo, hi))
                p = np.exp(x - x.max())
                out[row, h] = (p / p.sum()) @ v[lo:hi]
    return out


def attn_wide(c):
    """attn() for many rows: one matrix of scores for each sequence and head."""
    H, KV, D = c["n_head"], c["n_kv"], c["D"]
    out = np.full((c["n_rows"], H, D), np.nan)
    for s in range(c["n_seq"]):
        n, row = int(c["nq"][s]), int(c["q_start"][s])
        if not n:
            continue
        pos, lo, hi = (np.asarray(x)[:, None] for x in zip(*[row_range(c, s, t, row + t) for t in range(n)]))
        for g in range(KV):
            k, v = c["k"][s, :int(c["kv_len"][s]), g], c["v"][s, :int(c["kv_len"][s]), g]
            if c["n_shared"]:
                k, v = np.concatenate([c["pk"][:, g], k]), np.concatenate([c["pv"][:, g], v])
            j = np.arange(len(k))
            seen = (j >= lo) & (j < hi)
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                x = c["scale"] * (c["q"][row:row + n, h].astype(np.float64) @ k.T)
                if c["softcap"]:
                    x = c["softcap"] * np.tanh(x / c["softcap"])
                if c["slopes"] is not None:
                    x = x - float(c["slopes"][h]) * np.abs(pos - j)
                x = np.where(seen, x, -np.inf)
                top = x.max(axis=1, keepdims=True, initial=-np.inf)
                p = np.exp(x - np.where(np.isfinite(top), top, 0.0))
                total = p.sum(axis=1, keepdims=True)
                out[row:row + n, h] = (p / np.where(total > 0, total, 1.0)) @ v
    return out


def make(rng, n_seq, nq, kv_len, max_kv, n_head, n_kv, D, t, causal=True, softcap=0.0, alibi=False, prefix=None,
         docs=None, n_shared=0, lead=0, tail=0, std=1.3, max_q=None):
    """A random call: `lead` and `tail` packed rows that belong to no sequence."""
    nq, kv_len = np.asarray(nq), np.asarray(kv_len)
    n_rows = lead + int(nq.sum()) + tail
    c = {"n_seq": n_seq, "nq": nq, "kv_len": kv_len, "max_kv": max_kv, "n_head": n_head, "n_kv": n_kv, "D": D, "t": t,
         "causal": causal, "softcap": softcap, "n_shared": n_shared, "n_rows": n_rows, "scale": 1 / np.sqrt(D),
         "max_q": int(nq.max()) if max_q is None else max_q}
    c["scale"] = float(np.float32(c["scale"]))
    c["q_start"] = lead + np.concatenate([[0], np.cumsum(nq)])
    c["q"] = (rng.standard_normal((n_rows, n_head, D)) * std).astype(np.float32)
    for n, shape in (("k", (n_seq, max_kv, n_kv, D)), ("v", (n_seq, max_kv, n_kv, D)),
                     ("pk", (n_shared, n_kv, D)), ("pv", (n_shared, n_kv, D))):
        c[n + "_raw"], c[n] = to_cache(rng.standard_normal(shape), t)
    c["slopes"] = (2.0 ** (-8.0 * np.arange(1, n_head + 1) / n_head)).astype(np.float32) if alibi else None
    c["prefix_len"] = None if prefix is None else np.asarray(prefix)
    c["doc_start"], c["doc_end"] = (None, None) if docs is None else docs(c)
    return c


def run(hip, c, shared=None, out=None, k=None, v=None, strides=None, keep_out=None):
    """The call on the device: out as numpy."""
    shared = c["n_shared"] > 0 if shared is None else shared
    i32 = lambda a: None if a is None else hip.to_device(np.asarray(a, np.int32))  # noqa: E731
    D, KV = c["D"], c["n_kv"]
    st = strides or (c["max_kv"] * KV * D, KV * D, D)
    plain = c["q_start"][0] == 0 and c["n_rows"] == c["n_seq"] and (c["nq"] == 1).all()
    d = hip.attn_desc(c["t"], c["n_head"], KV, D, n_seq=c["n_seq"], n_rows=c["n_rows"], max_q=c["max_q"],
                      max_kv=c["max_kv"], q_start=None if plain and c.get("no_start") else i32(c["q_start"]),
                      kv_len=i32(c["kv_len"]), kv_seq_stride=st[0], kv_row_stride=st[1], kv_head_stride=st[2],
                      scale=c["scale"], causal=c["causal"], softcap=c["softcap"],
                      slopes=None if c["slopes"] is None else hip.to_device(c["slopes"]),
                      prefix_len=i32(c["prefix_len"]), doc_start=i32(c["doc_start"]), doc_end=i32(c["doc_end"]))
    q = hip.to_device(c["q"])
    k = hip.to_device(c["k_raw"]) if k is None else k
    v = hip.to_device(c["v_raw"]) if v is None else v
    o = hip.to_device(np.full((c["n_rows"], c["n_head"], D), 777.0, np.float32)) if out is None else out
    if shared:
        p = hip.attn_prefix(c["n_shared"], hip.to_device(c["pk_raw"]), hip.to_device(c["pv_raw"]), row_stride=KV * D,
                            head_stride=D)
        hip.attn_shared(d, p, q, k, v, o)
    else:
        hip.attn(d, q, k, v, o)
    if keep_out is not None:
        keep_out.extend([d, q, k, v, o] + ([p] if shared else []))
    return o.download(np.float32, c["n_rows"] * c["n_head"] * D).reshape(c["n_rows"], c["n_head"], D)


def tolerance(c):
    """Relative 2-norm error of a row that the arithmetic may have.

    A weight p is off by the error of its score in e-folds: the score's own
    rounding to fp32 in sums of D products (at most D 2^-24 |x|, about sqrt(D)
    of it), and for fp16 caches the cut of q to 22 bits, 2^-21 of each product.
    Scores here stay under 8 in 2-norm terms (|x| <= 8 std), a cap adds 2e-7
    cap. p's own cut adds 2^-21, the sums and exp2 a few 2^-23."""
    cut = {K.F32: 0.0, K.F16: 2.0 ** -21, K.BF16: 0.0}[c["t"]]
    x = 8.0 * float(np.abs(c["q"][np.isfinite(c["q"])]).std() * 1.7)
    return x * (cut + 12 * 2.0 ** -24) + cut + 2e-7 * c["softcap"] + 16 * 2.0 ** -23


def compare(c, got, want):
    """Rows that a sequence serves within tolerance(), the others untouched."""
    none = np.isnan(want).all(axis=(1, 2))
    assert np.array_equal(got[none], np.full_like(got[none], 777.0)), "rows of no sequence were written"
    g, w = got[~none].astype(np.float64), want[~none]
    zero = (w == 0).all(axis=2)
    assert (g[zero] == 0).all(), "rows that see nothing"
    err = np.linalg.norm(g - w, axis=2)
    rel = err / np.maximum(np.linalg.norm(w, axis=2), 1e-30)
    worst = rel[~zero].max() if (~zero).any() else 0.0
    assert worst <= tolerance(c), (worst, tolerance(c))


def append(c, k_new, v_new, n_rot, base, interleaved, pos0, eps, qw, kw):
    """(q_out, k, v) in 64 bits: rows and caches after the step."""
    def turn(x, w, pos):
        x = x.astype(np.float64)
        if w is not None:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * w
        y = x.copy()
        i = np.arange(n_rot // 2)
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n_rot // 2)
        ang = (pos + pos0) * float(np.float32(base)) ** (-2.0 * i / max(n_rot, 1))
        y[..., a] = x[..., a] * np.cos(ang) - x[..., b] * np.sin(ang)
        y[..., b] = x[..., a] * np.sin(ang) + x[..., b] * np.cos(ang)
        return y
    q, k, v = np.full(c["q"].shape, np.nan), c["k"].copy(), c["v"].copy()
    stored = np.zeros(c["k"].shape[:2], bool)
    for s in range(c["n_seq"]):
        for t in range(int(c["nq"][s])):
            row, pos = int(c["q_start"][s]) + t, int(c["kv_len"][s]) - int(c["nq"][s]) + t
            q[row] = turn(c["q"][row], qw, pos)
            if 0 <= pos < c["max_kv"]:
                k[s, pos], v[s, pos], stored[s, pos] = turn(k_new[row], kw, pos), v_new[row], True
    return q, k, v, stored
