"""The attention of a decode chain as cases that can be timed: the softmax
attention of query rows over their sequences' caches, the same for a batch
whose sequences share one long prefix, and the step before it that norms,
rotates and stores new rows in the caches.

One row of queries is [n_head][head_dim] fp32, as the projections give it; a
cache is [sequence][row][n_kv_head][head_dim] in fp32 (the engine's own),
fp16 or bf16. Rows of all sequences are packed one behind the other, a
sequence's rows being its newest positions. `own` says whether run() calls
the library (katali-lab_amd/katali_hip.py) or the plain form below.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False
DEV = "cuda"
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
GGML = {"f32": 0, "f16": 1, "bf16": 30}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------
def case(name, op, seqs, heads, kv_heads, dim, cache, rows, keys, **more):
    c = {"name": name, "op": op, "seqs": seqs, "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": cache,
         "rows": rows, "keys": keys, "ragged": False, "causal": True, "softcap": 0.0, "alibi": False, "prefix": 0,
         "docs": 0, "shared": 0, "n_rot": 0, "interleaved": False, "norm": False}
    c.update(more)
    return c


def listed():
    return [
        # one token of one conversation over the engine's own fp32 cache, early
        # in the context: a launch's latency is most of it
        case("attn_token_f32_300", "attn", 1, 32, 8, 128, "f32", 1, 300),
        # one token deep in a long document, fp16 cache: half a gigabyte of keys and values
        case("attn_token_f16_131072", "attn", 1, 32, 8, 128, "f16", 1, 131072),
        # one token each of 32 requests of mixed lengths, scores biased by
        # distance, eight query heads to a key head
        case("attn_batch_bf16_4096_bias", "attn", 32, 32, 4, 128, "bf16", 1, 4096, ragged=True, alibi=True),
        # a whole prompt of packed documents, its last rows padding that sees nothing
        case("attn_prompt_f16_4096_docs", "attn", 1, 32, 8, 128, "f16", 4096, 4096, docs=6),
        # five prompts of odd lengths with a two-sided prefix each, capped scores, wide heads
        case("attn_prompts_bf16_1531_cap_prefix", "attn", 5, 16, 2, 256, "bf16", 1531, 1531, ragged=True,
             softcap=50.0, prefix=400),
        # the next 509 tokens of a prompt read in pieces, behind 15 thousand, biased by distance
        case("attn_piece_f16_16000_bias", "attn", 1, 32, 8, 128, "f16", 509, 16000, alibi=True),
        # a prompt over the engine's own fp32 cache, narrow heads, capped scores
        case("attn_prompt_f32_1000_cap", "attn", 1, 24, 8, 64, "f32", 1000, 1000, softcap=30.0),
        # four requests right behind a short common instruction
        case("shared_f16_4x1000", "shared", 4, 32, 8, 128, "f16", 1, 40, ragged=True, shared=1000),
        # 64 requests about one long common document
        case("shared_bf16_64x16384", "shared", 64, 32, 8, 128, "bf16", 1, 1024, ragged=True, shared=16384),
        # nine requests of a few drafted tokens each, capped scores and a bias by distance
        case("shared_f16_9x5003_cap_bias", "shared", 9, 16, 16, 64, "f16", 5, 300, ragged=True, shared=5003,
             softcap=30.0, alibi=True),
        # the step before attention, one token
        case("append_token_f32", "append", 1, 32, 8, 128, "f32", 1, 300, n_rot=128, norm=True),
        # the step before attention, three prompts of up to 2049 tokens, half of each head rotated
        case("append_prompts_f16_2049", "append", 3, 16, 2, 256, "f16", 2049, 4100, ragged=True, n_rot=128, norm=True),
    ]


def log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attn", "attn", "attn", "shared", "shared", "append"])
    dim = rng.choice([64, 128, 128, 256])
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 2, 3, 4, 5, 8])
    cache = rng.choice(["f32", "f16", "bf16"])
    more = {"ragged": rng.random() < 0.7, "softcap": rng.choice([0.0, 0.0, 30.0, 50.0]), "alibi": rng.random() < 0.4}
    if op == "append":
        seqs, rows = rng.randint(1, 6), log_size(rng, 1, 1500)
        keys = rows + log_size(rng, 1, 3000)
        more.update(softcap=0.0, alibi=False, n_rot=rng.choice([dim, dim // 2]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.6)
    elif op == "shared":
        seqs, rows = log_size(rng, 2, 40), rng.choice([1, 1, 1, 2, 7])
        keys = rows + log_size(rng, 1, 700)
        more.update(shared=log_size(rng, 17, 9000))
    elif rng.random() < 0.5:   # tokens
        seqs = log_size(rng, 1, 24)
        rows = 1
        keys = log_size(rng, 1, 60000 // seqs)
        more.update(docs=rng.choice([0, 0, 3]))
    else:                      # prompts and pieces of them
        seqs = rng.randint(1, 4)
        rows = log_size(rng, 2, 1500)
        keys = rows + rng.choice([0, 0, log_size(rng, 1, 2000)])
        more.update(docs=rng.choice([0, 0, 4]), prefix=rng.choice([0, 0, log_size(rng, 1, rows)]),
                    causal=rng.random() < 0.85)
    c = case("", op, seqs, heads, kv, dim, cache, rows, keys, **more)
    del c["name"]
    return c


def lengths(c):
    """(query rows, own keys) of each sequence; a case's, whatever its values."""
    rng = random.Random("%(seqs)d %(rows)d %(keys)d %(heads)d %(shared)d" % c)
    nq, nk = [], []
    for s in range(c["seqs"]):
        q = c["rows"] if s == 0 or not c["ragged"] else rng.randint(1, c["rows"])
        nq.append(q)
        nk.append(c["keys"] if s == 0 or not c["ragged"] else rng.randint(max(q, c["keys"] // 5), c["keys"]))
    return nq, nk


def ranges(c):
    """Of each packed row: its sequence, its position, and the first and the
    one past the last key that its masks leave, as arrays."""
    nq, nk = lengths(c)
    rng = random.Random("docs %(seqs)d %(rows)d %(keys)d" % c)
    sh = c["shared"]
    seq = np.repeat(np.arange(c["seqs"]), nq)
    pos = np.concatenate([np.arange(k - q, k) for q, k in zip(nq, nk)]) + sh
    end = np.asarray(nk)[seq] + sh
    pre = np.asarray([rng.randint(c["prefix"] // 2, c["prefix"]) if c["prefix"] else 0 for _ in nk])
    lo, hi = np.zeros_like(pos), end.copy()
    if c["causal"]:
        hi = np.minimum(hi, np.maximum(pos + 1, pre[seq]))
    d0, d1 = np.zeros_like(pos), np.full_like(pos, 1 << 30)
    if c["docs"]:
        at = 0
        for q, k in zip(nq, nk):
            cuts = np.asarray([0] + sorted(rng.randint(1, max(1, k - 1)) for _ in range(c["docs"] - 1)) + [1 << 30])
            which = np.searchsorted(cuts, pos[at:at + q], side="right")
            d0[at:at + q], d1[at:at + q] = cuts[which - 1], cuts[which]
            if q > 8:   # a prompt's last three rows are padding: no key at all
                d0[at + q - 3:at + q] = d1[at + q - 3:at + q] = 0
            at += q
    return seq, pos, np.maximum(lo, d0), np.minimum(hi, d1), pre, d0, d1


def work(c):
    nq, nk = lengths(c)
    width = {"f32": 4, "f16": 2, "bf16": 2}[c["cache"]]
    row_q, row_kv = 4 * c["heads"] * c["dim"], 2 * width * c["kv_heads"] * c["dim"]
    if c["op"] == "append":
        new = sum(nq)
        return {"bytes": new * (2 * row_q + 2 * 4 * c["kv_heads"] * c["dim"] + row_kv),
                "flops": new * (c["heads"] + c["kv_heads"]) * c["dim"] * 6}
    seq, _, lo, hi, _, _, _ = ranges(c)
    pairs = int(np.maximum(hi - lo, 0).sum())
    # keys that some row sees: from the first to the last of each sequence
    seen = 0
    for s in range(c["seqs"]):
        m = (seq == s) & (hi > lo)
        if m.any():
            seen += max(0, int(hi[m].max()) - max(int(lo[m].min()), c["shared"]))
    return {"bytes": sum(nq) * 2 * row_q + (seen + c["shared"]) * row_kv, "flops": 4 * pairs * c["heads"] * c["dim"]}


# ---------------------------------------------------------------------------
# the inputs
# ---------------------------------------------------------------------------
def inputs(c, seed):
    """The values, made in one order from the seed alone."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.randn(*shape, device=DEV, generator=g) * std

    H, KV, D, t = c["heads"], c["kv_heads"], c["dim"], TYPES[c["cache"]]
    n = sum(lengths(c)[0])
    # scores of about unit deviation; several times that where they are capped
    v = {"q": normal(n, H, D, std=4.0 if c["softcap"] else 1.3),
         "k": normal(c["seqs"], c["keys"], KV, D).to(t), "v": normal(c["seqs"], c["keys"], KV, D).to(t)}
    if c["shared"]:
        v["pk"], v["pv"] = normal(c["shared"], KV, D).to(t), normal(c["shared"], KV, D).to(t)
    if c["op"] == "append":
        v["nk"], v["nv"] = normal(n, KV, D, std=2.0), normal(n, KV, D)
        if c["norm"]:
            v["qw"], v["kw"] = 1.0 + normal(D, std=0.1), 1.0 + normal(D, std=0.1)
    return v


def prepare(c, seed):
    s = {"case": dict(c), **inputs(c, seed)}
    nq, nk = lengths(c)
    seq, pos, _, _, pre, d0, d1 = ranges(c)
    start = np.concatenate([[0], np.cumsum(nq)])

    def dev(a, t=torch.int32):
        return torch.as_tensor(np.asarray(a), dtype=t).to(DEV)

    s["q_start"], s["kv_len"] = dev(start), dev(nk)
    s["prefix_len"] = dev(pre) if c["prefix"] else None
    s["doc_start"], s["doc_end"] = (dev(d0), dev(d1)) if c["docs"] else (None, None)
    s["slopes"] = dev(2.0 ** (-8.0 * np.arange(1, c["heads"] + 1) / c["heads"]), torch.float32) if c["alibi"] else None
    s["out"] = torch.zeros_like(s["q"])
    # packed rows to a rectangle [sequence][row] and back, and the rows' places
    t = np.arange(c["rows"])
    s["to_pad"] = dev(np.minimum(start[:-1, None] + t, start[-1] - 1), torch.int64)
    s["to_packed"] = dev(seq * c["rows"] + np.arange(len(seq)) - start[seq], torch.int64)
    s["pos_pad"] = dev(np.asarray(nk)[:, None] - np.asarray(nq)[:, None] + t + c["shared"], torch.int64)
    s["seq"], s["row"] = dev(seq, torch.int64), dev(pos - c["shared"], torch.int64)
    return s


# ---------------------------------------------------------------------------
# the plain form
# ---------------------------------------------------------------------------
def plain_attn(s):
    c = s["case"]
    S, H, KV, D, R, sh = c["seqs"], c["heads"], c["kv_heads"], c["dim"], c["rows"], c["shared"]
    G = H // KV
    q = s["q"][s["to_pad"]].view(S, R, KV, G, D).permute(0, 2, 3, 1, 4).reshape(S, KV, G * R, D)
    kt = s["k"].permute(0, 2, 3, 1).to(torch.float32, memory_format=torch.contiguous_format)
    sc = torch.matmul(q, kt.contiguous())
    if sh:
        pkt = s["pk"].permute(1, 2, 0).to(torch.float32, memory_format=torch.contiguous_format).contiguous()
        psc = torch.matmul(q.transpose(0, 1).reshape(KV, S * G * R, D), pkt)
        sc = torch.cat([psc.view(KV, S, G * R, sh).transpose(0, 1), sc], dim=-1)
    L = sc.shape[-1]
    sc = sc.view(S, KV, G, R, L) * (1.0 / math.sqrt(D))
    if c["softcap"]:
        sc = c["softcap"] * torch.tanh(sc / c["softcap"])
    j = torch.arange(L, device=DEV)
    pos = s["pos_pad"].view(S, 1, 1, R, 1)
    if c["alibi"]:
        sc = sc - s["slopes"].view(1, KV, G, 1, 1) * (pos - j).abs()
    vis = j < (s["kv_len"] + sh).view(S, 1, 1, 1, 1)
    if c["causal"]:
        upto = pos + 1
        if c["prefix"]:
            upto = torch.maximum(upto, s["prefix_len"].view(S, 1, 1, 1, 1))
        vis = vis & (j < upto)
    if c["docs"]:
        vis = vis & (j >= s["doc_start"][s["to_pad"]].view(S, 1, 1, R, 1))
        vis = vis & (j < s["doc_end"][s["to_pad"]].view(S, 1, 1, R, 1))
    sc = sc.masked_fill(~vis, -math.inf)
    m = sc.amax(dim=-1, keepdim=True)
    p = torch.exp(sc - torch.where(m > -math.inf, m, torch.zeros_like(m)))
    total = p.sum(dim=-1, keepdim=True)
    p = (p / torch.where(total > 0, total, torch.ones_like(total))).view(S, KV, G * R, L)
    v = s["v"].permute(0, 2, 1, 3).to(torch.float32, memory_format=torch.contiguous_format).contiguous()
    o = torch.matmul(p[..., sh:].contiguous(), v)
    if sh:
        pv = s["pv"].permute(1, 0, 2).to(torch.float32, memory_format=torch.contiguous_format).contiguous()
        pp = p[..., :sh].transpose(0, 1).reshape(KV, S * G * R, sh)
        o = o + torch.matmul(pp, pv).view(KV, S, G * R, D).transpose(0, 1)
    o = o.view(S, KV, G, R, D).permute(0, 3, 1, 2, 4).reshape(S * R, H, D)
    return o[s["to_packed"]]


def plain_rows(x, w, cos, sin, c):
    """One kind of rows through the head norm (w given) and the rotation."""
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + EPS) * w
    n = c["n_rot"]
    if c["interleaved"]:
        a, b = x[..., 0:n:2], x[..., 1:n:2]
    else:
        a, b = x[..., :n // 2], x[..., n // 2:n]
    ra, rb = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([ra, rb], dim=-1).flatten(-2) if c["interleaved"] else torch.cat([ra, rb], dim=-1)
    return torch.cat([turned, x[..., n:]], dim=-1)


def plain_append(s):
    c = s["case"]
    half = torch.arange(c["n_rot"] // 2, device=DEV, dtype=torch.float64)
    # the angles in 64 bits: far positions times small frequencies
    ang = s["row"].double().view(-1, 1, 1) * torch.exp2(half * (-2.0 * math.log2(1e6) / c["n_rot"]))
    cos, sin = torch.cos(ang).float(), torch.sin(ang).float()
    q = plain_rows(s["q"], s.get("qw"), cos, sin, c)
    k = plain_rows(s["nk"], s.get("kw"), cos, sin, c)
    s["k"][s["seq"], s["row"]] = k.to(s["k"].dtype)
    s["v"][s["seq"], s["row"]] = s["nv"].to(s["v"].dtype)
    return q


# ---------------------------------------------------------------------------
# the library's calls
# ---------------------------------------------------------------------------
class Buf:
    """A torch tensor on the GPU as the binding's buffers: it reads .ptr."""

    def __init__(self, t):
        self.t, self.ptr = t, t.data_ptr()


def buf(t):
    return None if t is None else Buf(t)


_hip = None


def hip():
    """The library through its Python binding."""
    global _hip
    if _hip is None:
        sys.path.insert(0, os.path.join(os.getcwd(), "katali-lab_amd"))
        import katali_hip
        _hip = katali_hip.KataliHip()
        if not _hip.probe():
            raise RuntimeError(_hip.status())
    return _hip


def plan(s):
    """The descriptor that a program keeps with its buffers."""
    if "plan" not in s:
        c, h = s["case"], hip()
        KV, D = c["kv_heads"], c["dim"]
        d = h.attn_desc(GGML[c["cache"]], c["heads"], KV, D, n_seq=c["seqs"], n_rows=s["q"].shape[0],
                        max_q=c["rows"], max_kv=c["keys"], q_start=buf(s["q_start"]), kv_len=buf(s["kv_len"]),
                        kv_seq_stride=c["keys"] * KV * D, kv_row_stride=KV * D, kv_head_stride=D,
                        scale=1.0 / math.sqrt(D), causal=c["causal"], softcap=c["softcap"], slopes=buf(s["slopes"]),
                        prefix_len=buf(s["prefix_len"]), doc_start=buf(s["doc_start"]), doc_end=buf(s["doc_end"]))
        more = None
        if c["shared"]:
            more = h.attn_prefix(c["shared"], buf(s["pk"]), buf(s["pv"]), row_stride=KV * D, head_stride=D)
        if c["op"] == "append":
            more = h.rope(c["n_rot"], 1e6, interleaved=c["interleaved"], eps=EPS, q_norm_w=buf(s.get("qw")),
                          k_norm_w=buf(s.get("kw")))
        s["plan"] = (d, more, {n: buf(s[n]) for n in ("q", "k", "v", "nk", "nv", "out") if n in s})
    return s["plan"]


def run(s):
    c = s["case"]
    if own:
        d, more, b = plan(s)
        if c["op"] == "attn":
            hip().attn(d, b["q"], b["k"], b["v"], b["out"])
        elif c["op"] == "shared":
            hip().attn_shared(d, more, b["q"], b["k"], b["v"], b["out"])
        else:
            hip().kv_append(d, more, b["q"], b["nk"], b["nv"], b["out"], b["k"], b["v"])
        return [s["out"], s["k"], s["v"]] if c["op"] == "append" else [s["out"]]
    if c["op"] == "append":
        return [plain_append(s), s["k"], s["v"]]
    return [plain_attn(s)]


# ---------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------
def exact_append(c, v):
    nq, nk = lengths(c)
    n = c["n_rot"]
    k, w = v["k"].double(), v["v"].double()
    q_out, at = torch.empty_like(v["q"], dtype=torch.float64), 0

    def rows(x, weight, p):
        x = x.double()
        if weight is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) * weight.double()
        i = torch.arange(n // 2, device=DEV)
        first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + n // 2)
        turn = torch.polar(torch.ones(len(p), n // 2, dtype=torch.float64, device=DEV),
                           p[:, None].double() * (1e6 ** (-2.0 * i.double() / n)))[:, None]
        z = torch.complex(x[..., first], x[..., second]) * turn
        y = x.clone()
        y[..., first], y[..., second] = z.real, z.imag
        return y

    for b in range(c["seqs"]):
        p = torch.arange(nk[b] - nq[b], nk[b], device=DEV)
        q_out[at:at + nq[b]] = rows(v["q"][at:at + nq[b]], v.get("qw"), p)
        k[b, p] = rows(v["nk"][at:at + nq[b]], v.get("kw"), p)
        w[b, p] = v["nv"][at:at + nq[b]].double()
        at += nq[b]
    return [q_out, k, w]


def exact(c, seed):
    v = inputs(c, seed)
    if c["op"] == "append":
        return exact_append(c, v)
    nq, nk = lengths(c)
    _, pos, lo, hi, _, _, _ = ranges(c)
    H, KV, D, sh = c["heads"], c["kv_heads"], c["dim"], c["shared"]
    out, at = torch.zeros_like(v["q"], dtype=torch.float64), 0
    for b in range(c["seqs"]):
        n = nq[b]
        first, last, p = (torch.as_tensor(x[at:at + n]).to(DEV)[:, None] for x in (lo, hi, pos))
        for g in range(KV):
            k, w = v["k"][b, :nk[b], g].double(), v["v"][b, :nk[b], g].double()
            if sh:
                k, w = torch.cat([v["pk"][:, g].double(), k]), torch.cat([v["pv"][:, g].double(), w])
            j = torch.arange(len(k), device=DEV)
            hidden = (j < first) | (j >= last)
            for h in range(g * (H // KV), (g + 1) * (H // KV)):
                x = v["q"][at:at + n, h].double() @ k.T.contiguous() / math.sqrt(D)
                if c["softcap"]:
                    x = c["softcap"] * torch.tanh(x / c["softcap"])
                if c["alibi"]:
                    x = x - float(np.float32(2.0 ** (-8.0 * (h + 1) / H))) * (p - j).abs()
                x = torch.softmax(x.masked_fill(hidden, -1e300), dim=-1).masked_fill(hidden, 0.0)
                out[at:at + n, h] = x @ w
        at += n
    return [out]
