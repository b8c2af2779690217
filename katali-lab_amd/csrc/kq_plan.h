// kq_plan.h — host-side launch decisions that need no device, shared by the
// launchers and by CPU tests (plain C++, no HIP headers).
#pragma once

#include <stdint.h>

#include <initializer_list>

namespace kq {

// The one-launch layers (the XCD-sliced layer and its stack) wait between
// their workgroups, so all `grid` of them must be resident at once: one per
// CU on a device of exactly `grid` CUs (the slot-to-XCD mapping), with the
// occupancy API's blocks_per_cu for the kernel's block size and LDS at
// least 1.
inline bool xcd_coresident(int cus, int blocks_per_cu, uint32_t grid) {
    return cus > 0 && (uint32_t)cus == grid && blocks_per_cu >= 1 && (uint64_t)blocks_per_cu * (uint64_t)cus >= grid;
}

// Kernel A: units of 32 h values (a q8_1 block) put ceil(units / cus) on the
// busiest CU; half units put ceil(2 units / cus) halves there. Half units when
// that is less work on the busiest CU and the units pair up by eights (384
// units on 256 CUs: 2 against 1.5).
inline bool half_units(uint32_t units, uint32_t cus) {
    if (!cus || units % 8) return false;
    const uint64_t full = (units + cus - 1) / cus, half = (2ull * units + cus - 1) / cus;
    return half < 2 * full;
}

// gfx950's LDS per workgroup
constexpr uint32_t LDS_PER_WG = 160 * 1024;

// The wide down projection's launch (k_moe_down_wide): a workgroup of nw waves
// takes rpw output rows of all slots, S lanes per (slot, row) pair and N items
// per lane and batch. h in item order is 352 bytes per block in tiles of 16
// items, each slot from a tile of its own while that fits, else slot after slot
// (pack): at most 1056 bytes more than the 11/8 per value of the layer's LDS
// rule, which keeps 2116 bytes for the rows' sums, so every shape that rule
// admits has a plan.
constexpr uint32_t DW_SLOTS = 17;       // the most slots of a layer (16 routed and the shared expert)
constexpr uint32_t DW_MAX_ROWS = 200;   // inv_rpw exact, a thread per row at the end
struct DownPlan {
    uint32_t S, N, rpw, inv_rpw, nw, lds;
    bool pack;
};
inline uint32_t item_tile_bytes(uint32_t items, uint32_t ipb) { return (items + 15) / 16 * (16 / ipb * 352); }
inline bool down_plan(bool q6, uint32_t hidden, uint32_t ffn, uint32_t n_slots, uint32_t cus, DownPlan &p) {
    const uint32_t ipb = q6 ? 4 : 8, nb = ffn / 256, items = nb * ipb, nmax = q6 ? 4 : 8;
    if (!cus || nb <= 4 || n_slots == 0 || n_slots > DW_SLOTS) return false;
    // rows of 5 to 16 blocks: four block columns of lanes; longer rows: the
    // whole wave (the grouped down kernels' split)
    p.S = nb > 16 ? 64 : 4 * ipb;
    const uint32_t steps = (items + p.S - 1) / p.S, batches = (steps + nmax - 1) / nmax;
    p.N = (steps + batches - 1) / batches;
    // two workgroups of 8 waves per CU while their h fits twice, with Q4_K up
    // to 7/16 of the LDS (nine slots of 6144: 41.9 us staged twice, 40.5 once),
    // else one of 16 waves; never more waves than the rows give pairs
    uint32_t hb = n_slots * item_tile_bytes(items, ipb);
    const uint32_t per_cu = hb + (q6 ? 4096 : 10240) <= LDS_PER_WG / 2 ? 2 : 1, wmax = per_cu == 2 ? 8 : 16;
    p.rpw = (hidden + per_cu * cus - 1) / (per_cu * cus);
    const uint32_t most_rpw = p.rpw < DW_MAX_ROWS ? p.rpw : DW_MAX_ROWS;
    p.pack = hb + (most_rpw * n_slots + DW_SLOTS) * 4 > LDS_PER_WG;
    if (p.pack) hb = item_tile_bytes(n_slots * items, ipb);
    if (hb + (n_slots + DW_SLOTS) * 4 > LDS_PER_WG) return false;
    const uint32_t fit = ((LDS_PER_WG - hb) / 4 - DW_SLOTS) / n_slots;
    for (uint32_t most : {fit, DW_MAX_ROWS})
        if (p.rpw > most) p.rpw = most;
    p.inv_rpw = ((1u << 20) + p.rpw - 1) / p.rpw;
    p.nw = (p.rpw * n_slots + 64 / p.S - 1) / (64 / p.S);
    p.nw = p.nw < 4 ? 4 : (p.nw > wmax ? wmax : p.nw);
    p.lds = hb + (p.rpw * n_slots + DW_SLOTS) * 4;
    return true;
}

// How an attention call's rows and keys are spread over workgroups. The rows
// of one key head of a sequence (query rows x the heads that share the key
// head) make tiles: of 16 where they are few (the waves of a workgroup share
// the rows and divide the keys), else of 64 or 128, 16 or 32 to a wave, which
// walk the same keys together. Keys are split where the tiles alone would leave
// CUs idle; the parts' sums meet in `slots` partial results of each row
// (0: one part, written as the output). A shared prefix is either an item of
// its own for the rows of all sequences together (shared_tiles > 0), or
// walked by each sequence's items ahead of its own keys.
enum AttnForm { ATTN_ROWS, ATTN_TILES, ATTN_MIXED };   // MIXED: pooled rows in tiles, own ones few
struct AttnPlan {
    AttnForm form;
    uint32_t own_tiles, own_splits, own_items;
    uint32_t shared_tiles, shared_splits, shared_items;
    uint32_t slots, own_chunk, shared_chunk;   // chunk: keys that are worth a part of their own
};
constexpr uint32_t ATTN_MAX_SLOTS = 64;
constexpr uint64_t ATTN_SCRATCH = 64ull << 20;   // partial results: head_dim sums, a maximum and a sum each
constexpr uint32_t ATTN_FEW_ROWS = 32;           // rows of a key head: up to here a sequence's rows are pooled over a shared
                                                 // prefix, and a pool of more takes wide tiles
constexpr int ATTN_F32 = 0, ATTN_F16 = 1, ATTN_BF16 = 30;   // cache types (ggml ids)
// Rows of a workgroup's tile: 16 or 32 for each of four or eight waves, by what registers and LDS hold.
constexpr int attn_tile_rows(int type, int head_dim) {
    return (type == ATTN_F32 && head_dim != 128) || (type == ATTN_F16 && head_dim == 256) ||
                   (type == ATTN_BF16 && head_dim == 128) ? 64 : 128;
}
// Whether one kernel takes a shared prefix's tiles beside the rows of each sequence, else two launches do.
constexpr bool attn_mixed(int type, int head_dim) { return head_dim == 64 || (head_dim == 128 && type != ATTN_F32); }

inline AttnPlan attn_plan(uint32_t n_seq, uint32_t n_rows, uint32_t max_q, uint32_t n_kv, uint32_t group,
                          uint32_t max_kv, uint32_t n_shared, uint32_t head_dim, int type, uint32_t cus) {
    const bool f32 = type == ATTN_F32;
    AttnPlan p = {};
    const uint64_t per_seq = (uint64_t)max_q * group, n_head = (uint64_t)n_kv * group;
    const uint64_t most_slots = ATTN_SCRATCH / ((uint64_t)n_rows * n_head * (head_dim + 2) * 4);
    const uint32_t cap = most_slots < ATTN_MAX_SLOTS ? (uint32_t)most_slots : ATTN_MAX_SLOTS;
    const uint32_t waves = 4;                               // ROWS_WAVES
    const uint32_t few = waves * (f32 ? 16 : 32);           // a tile of keys for every wave
    const uint32_t many = f32 ? 64 : 128;                  // two stages or more
    auto cover = [](uint64_t n, uint64_t by) { return (n + by - 1) / by; };
    // parts for `items` items of up to `keys` keys each, so that about `want` workgroups come of it;
    // a part has at least `least` keys, and shorter items take fewer parts of the same length
    auto split = [&](uint64_t items, uint64_t keys, uint64_t want, uint32_t least, uint32_t most, uint32_t &parts,
                     uint32_t &chunk) {
        uint64_t n = want / (items ? items : 1);
        const uint64_t worth = cover(keys, least);
        n = n < worth ? n : worth;
        n = n < most ? n : most;
        parts = n < 1 ? 1 : (uint32_t)n;
        const uint64_t c = cover(keys ? keys : 1, parts);
        chunk = (uint32_t)(c > least ? c : least);
    };
    // Tiles of 16 rows read the keys once for each tile, but start sooner and spread
    // further: they win while the tiles times their keys are few for the CUs. Up to 16 rows
    // there is one tile. 32 heads over 8 of 128, 256 CUs, us with tiles of 16 / of 64 and more, fp16:
    // 64 rows over 4000 keys (512 thousand tile-keys) 30 / 39, 128 rows 47 / 45, 4 x 64 rows over
    // 1000 keys 25 / 35, over 4000 76 / 57; fp32: 32 rows over 4000 keys 35 / 41, 64 rows 57 / 49.
    auto few_for_cus = [&](uint64_t heads_rows, uint64_t n, uint64_t keys, uint64_t per_cu) {
        return cover(heads_rows, 16) * n * (keys ? keys : 1) <= per_cu * 128 / head_dim * cus;
    };
    // Workgroups for tiles of 16 rows: two for each CU; with 16-bit caches one where that fills the CUs
    // by 7/8 and 256-wide heads leave room for one only (3 tokens over 1600 keys of 8 heads 24 us
    // with two, 17 with one; 60 rows over 1000 28 / 22) or one part for each item is that already
    // (60 tokens over up to 9000 keys of 4 x 128 160 / 155 us; fp32 32 over 2000 of 8 x 128 62 / 67).
    auto rows_want = [&](uint64_t items) {
        const uint64_t n = cus / (items ? items : 1);
        return !f32 && n * items * 8 >= 7ull * cus && (head_dim == 256 || n == 1) ? cus : 2 * cus;
    };
    const uint64_t all_keys = (uint64_t)max_kv + n_shared;
    // Workgroups for wide tiles, of which a CU holds two: two for each CU. Tiles that fill the CUs once
    // and a part of them again are parted for four, else the second of a CU is alone with its keys for
    // half the time, where the join is worth it: with fp32 up to 7/4 of the CUs (24 heads of 64, 1000 rows
    // over 1000 keys, 376 tiles, 55 / 46 us; 528 rows over 2028, 264 tiles, 105 / 75), with 16 bits up to 3/2
    // and from 1500 keys on (fp16, 264 tiles of 128: 1056 rows over 1056 keys 53 / 56, over 2556 130 / 105,
    // over 5000 250 / 186). Of bf16 256 and fp32 128 a CU holds one: one for each CU where that fills them by
    // 7/8 (1000 rows of 8 heads over 2 of bf16 256, 1000 keys 62 / 46; 4000 115 / 96; fp32 128 46 / 34 and 101 / 93).
    auto tiles_want = [&](uint64_t items) {
        const bool alone = (f32 && head_dim == 128) || (type == ATTN_BF16 && head_dim == 256);
        const uint64_t n = cus / (items ? items : 1);
        if (alone) return n * items * 8 >= 7ull * cus ? cus : 2 * cus;
        return items > cus && (f32 ? items * 4 <= 7ull * cus : items * 2 <= 3ull * cus && all_keys >= 1500) ? 4 * cus : 2 * cus;
    };
    // keys over which four waves take as long as a join
    const uint64_t brief = (f32 ? 128 : 384) * 128 / head_dim;
    // (over so few keys a shared prefix is walked by each sequence: 40 over 100 + 100 keys 11 us against 15)
    const bool pool = n_shared && n_seq > 1 && per_seq <= ATTN_FEW_ROWS && cap >= 2 && all_keys > brief;
    const bool tiles = !pool && per_seq > 16 && !few_for_cus(per_seq, (uint64_t)n_seq * n_kv, all_keys, f32 ? 1400 : 3000);
    p.own_tiles = (uint32_t)cover(per_seq, tiles ? attn_tile_rows(type, (int)head_dim) : 16);
    const uint64_t own = (uint64_t)p.own_tiles * n_seq * n_kv;
    if (pool) {
        const uint64_t pooled = (uint64_t)n_rows * group;
        // the prefix for more than two tiles of 16 of all sequences' rows in wide tiles: 64 rows
        // over 2000 keys 17 us against 20, over 8000 22 / 26, 160 over 1000 19 / 21, 256 over 8000
        // 45 / 59 (but 96 rows over 4000 keys 28 / 22)
        p.form = pooled > ATTN_FEW_ROWS ? ATTN_MIXED : ATTN_ROWS;
        // (one launch's tiles are of 16 rows a wave)
        const uint32_t wide = attn_mixed(type, (int)head_dim) ? 16 * waves : (uint32_t)attn_tile_rows(type, (int)head_dim);
        p.shared_tiles = (uint32_t)cover(pooled, p.form == ATTN_MIXED ? wide : 16);
        const uint64_t shared = (uint64_t)n_kv * p.shared_tiles;
        const bool apart = !attn_mixed(type, (int)head_dim);   // two launches
        split(shared, n_shared, apart && p.form == ATTN_MIXED ? tiles_want(shared) : 2 * cus,
              p.form == ATTN_MIXED ? many : few, cap / 2, p.shared_splits, p.shared_chunk);
        split(own, max_kv, apart ? rows_want(own) : 2 * cus, few, cap - p.shared_splits, p.own_splits, p.own_chunk);
        p.slots = p.shared_splits + p.own_splits;
    } else {
        p.form = tiles ? ATTN_TILES : ATTN_ROWS;
        split(own, all_keys, tiles ? tiles_want(own) : rows_want(own), tiles ? many : few, cap, p.own_splits, p.own_chunk);
        // one part and no join where parts save less than the join costs, its price taken to grow with the
        // rows to be joined: of 8 x 128 fp16, 1 token over 300 keys 10.6 us with parts, 9.1 without (560: 10.6 / 11.7),
        // 20 over 1000 19.6 / 18.5, 32 over 600 19.7 / 17.4; fp32 1 over 130 10.3 / 10.0 (200: 10.4 / 11.4)
        if (!tiles && all_keys * (p.own_splits - 1) * 8 * cus <= brief * p.own_splits * 3 * (2 * cus + 8 * own))
            split(own, all_keys, 1, few, 1, p.own_splits, p.own_chunk);
        p.slots = p.own_splits > 1 ? p.own_splits : 0;
    }
    p.own_items = (uint32_t)(own * p.own_splits);
    p.shared_items = n_kv * p.shared_tiles * p.shared_splits;
    return p;
}

}  // namespace kq
