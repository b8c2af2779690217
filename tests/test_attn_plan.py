"""How an attention call's rows and keys are spread over workgroups
(attn_plan in katali-lab_amd/csrc/kq_plan.h), compiled with the host compiler
and swept here over head layouts, lengths, batches and CU counts; no device."""
import os
import subprocess

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(REPO, "katali-lab_amd", "csrc")

DRIVER = r"""
#include <stdio.h>
#include "kq_plan.h"
using namespace kq;
static unsigned long n, bad, forms[3], split, direct;
static void look(unsigned S, unsigned rows, unsigned max_q, unsigned kv, unsigned g, unsigned keys, unsigned sh,
                 unsigned D, int type, unsigned cus) {
    const AttnPlan p = attn_plan(S, rows, max_q, kv, g, keys, sh, D, type, cus);
    const unsigned long long per = (unsigned long long)max_q * g;
    const unsigned own_tile = p.form == ATTN_TILES ? attn_tile_rows(type, D) : 16;
    bool ok = p.own_splits >= 1 && p.own_chunk >= 1;
    ok = ok && (unsigned long long)p.own_tiles * own_tile >= per && (unsigned long long)(p.own_tiles - 1) * own_tile < per;
    ok = ok && (unsigned long long)S * kv * p.own_tiles * p.own_splits == p.own_items;
    ok = ok && (per > 16 || p.form != ATTN_TILES);
    if (p.shared_items) {
        const unsigned t = p.form == ATTN_ROWS ? 16 : attn_mixed(type, D) ? 64 : attn_tile_rows(type, D);
        ok = ok && sh && S > 1 && p.shared_chunk >= 1 && p.slots == p.own_splits + p.shared_splits;
        ok = ok && (unsigned long long)p.shared_tiles * t >= (unsigned long long)rows * g;
        ok = ok && kv * p.shared_tiles * p.shared_splits == p.shared_items;
    } else {
        ok = ok && p.form != ATTN_MIXED && p.slots == (p.own_splits > 1 ? p.own_splits : 0);
    }
    // partial results fit the scratch, and one lane of a wave holds one slot's maximum
    ok = ok && p.slots <= ATTN_MAX_SLOTS &&
         (unsigned long long)rows * kv * g * p.slots * (D + 2) * 4 <= ATTN_SCRATCH;
    // a chunk times the parts reaches over all keys (else the last keys had no part)
    const unsigned long long own_keys = p.shared_items ? keys : (unsigned long long)keys + sh;
    ok = ok && (unsigned long long)p.own_chunk * p.own_splits >= own_keys;
    if (p.shared_items) ok = ok && (unsigned long long)p.shared_chunk * p.shared_splits >= sh;
    n++, forms[p.form]++, split += p.slots > 0, direct += p.slots == 0;
    if (!ok) {
        if (bad++ < 5) printf("bad: S=%u rows=%u max_q=%u kv=%u g=%u keys=%u sh=%u D=%u type=%d cus=%u\n", S, rows, max_q, kv, g, keys, sh, D, type, cus);
    }
}
int main() {
    for (unsigned cus : {1u, 64u, 256u, 304u})
        for (int type : {ATTN_F32, ATTN_F16, ATTN_BF16})
            for (unsigned D : {64u, 128u, 256u})
                for (unsigned kv : {1u, 2u, 8u, 16u})
                    for (unsigned g : {1u, 3u, 4u, 16u, 40u})
                        for (unsigned S : {1u, 2u, 7u, 64u, 1000u, 65535u})
                            for (unsigned q : {1u, 2u, 9u, 200u, 4096u})
                                for (unsigned keys : {0u, 1u, 40u, 1000u, 131072u, 0x7FFFEFFFu - 20000u})
                                    for (unsigned sh : {0u, 1u, 17u, 20000u}) {
                                        if ((unsigned long long)S * q * kv * g > 0x7FFF0000ull) continue;
                                        look(S, S * q, q, kv, g, keys, sh, D, type, cus);
                                    }
    // the shapes that the GPU tests count on: keys in parts, a prefix walked by all rows together, wide tiles
    for (int type : {ATTN_F32, ATTN_F16, ATTN_BF16})
        for (unsigned D : {64u, 128u, 256u}) {
            const unsigned r = (D == 64 ? 900 : D == 128 ? 640 : 460) + 3;
            if (attn_plan(1, r, r, 8, 4, r, 0, D, type, 256).form != ATTN_TILES) bad++;
            if (attn_plan(4, 3, 1, 2, 4, 1900, 0, D, type, 256).own_splits < 2) bad++;
            if (attn_plan(4, 19, 9, 2, 7, 1900, 0, D, type, 256).own_splits < 2) bad++;
            const AttnPlan few = attn_plan(2, 1, 1, 2, 4, 300, 777, D, type, 256), many = attn_plan(9, 24, 3, 2, 4, 300, 790, D, type, 256);
            if (few.form != ATTN_ROWS || !few.shared_items || many.form != ATTN_MIXED) bad++;
        }
    printf("%lu %lu %lu %lu %lu %lu %lu\n", n, bad, forms[0], forms[1], forms[2], split, direct);
    return 0;
}
"""


def test_plans(tmp_path):
    src = tmp_path / "t.cpp"
    src.write_text(DRIVER)
    exe = tmp_path / "t"
    subprocess.run(["g++", "-std=c++17", "-O1", "-I" + CSRC, str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout
    n, bad, rows, tiles, mixed, split, direct = (int(x) for x in out.splitlines()[-1].split())
    assert bad == 0, out
    assert n > 10000 and min(rows, tiles, mixed, split, direct) > 100, out
