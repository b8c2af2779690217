// kq_attn.hip — softmax attention of query rows over their sequences' caches,
// and over a prefix that all sequences share.
//
//   x_j = scale (q . k_j);  x_j = cap tanh(x_j / cap) with a cap;
//   x_j -= slope_h |pos - j| with slopes;  o = sum_j p_j v_j, p = softmax over
//   the row's keys [lo, hi), where lo and hi come from the causal rule, the
//   two-sided prefix and the row's document. A row with no key gives zeros.
//
// One pass over the keys with a running maximum and sum (in log2 units). q
// and the outputs are fp32, and the matrix instructions take 16-bit operands
// with 16-bit caches, so q and p are each split into 16-bit terms, two of fp16
// (22 bits together) or three of bf16 (24), and each product is formed once per
// term into the same fp32 accumulators: nothing is rounded to 16 bits. (Two
// terms of bf16 were 2.5e-6 to 5.6e-6 off the definition in 64 bits, three are
// 2e-7 to 1.1e-6, as an fp32 evaluation is.) fp32 caches: the fp32 matrix
// instructions, and for many rows three bf16 terms of keys and values too.
//
// k_attn: a wave takes 16 rows (query rows x the heads of one key head), one
// row per lane column of the matrix tile, and walks its keys in tiles of 32
// (16 with fp32 caches). It computes S^T = K Q^T, so that a lane holds scores
// of one row only and row maxima need two cross-lane steps, and O^T = V^T P^T,
// whose B operand is P^T in the very registers that S^T came in: the keys of
// an operand may stand in any order if both operands have the same. V^T's
// operand wants four keys of one column in a lane; a lane loads 4 rows of V,
// D/16 columns each, and exchanges halves between them (v_perm), no LDS.
// k_attn_tile: the same for many rows, the keys staged through LDS.
#include <type_traits>

#include "kq_attn.h"

namespace kq {

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896341f;
constexpr float NEG_INF = -__builtin_inff();

template <class T, class S>
__device__ __forceinline__ T bits(const S &s) {
    static_assert(sizeof(T) == sizeof(S), "bits: sizes differ");
    T t;
    __builtin_memcpy(&t, &s, sizeof(T));
    return t;
}

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

// max / sum over the four lanes (one per 16-lane row) that hold one query row
__device__ __forceinline__ float rows_max(float v) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float rows_sum(float v) {
    v = swap_sum<16>(v, v);
    return swap_sum<32>(v, v);
}

// tanh to about 1e-7 of its value: below 1 the continued fraction
// u / (1 + u^2 / (3 + u^2 / (5 + u^2 / (7 + u^2 / 9)))), above it
// 1 - 2 / (e^2u + 1), both over one reciprocal. NaN stays NaN.
__device__ __forceinline__ float tanh_num(float u, float u2) { return u * fmaf(u2, u2 + 105.0f, 945.0f); }
__device__ __forceinline__ float tanh_den(float u2) { return fmaf(u2, fmaf(u2, 15.0f, 420.0f), 945.0f); }
__device__ __forceinline__ float tanh_below_1(float u) {
    const float u2 = u * u;
    return tanh_num(u, u2) * __builtin_amdgcn_rcpf(tanh_den(u2));
}
__device__ __forceinline__ float tanh_fast(float u) {
    const float u2 = u * u;
    const bool small = fabsf(u) < 1.0f;
    const float r = __builtin_amdgcn_rcpf(small ? tanh_den(u2) : exp2_hw(u * (2.0f * LOG2E)) + 1.0f);
    return small ? tanh_num(u, u2) * r : fmaf(-2.0f, r, 1.0f);
}

// Two fp32 values as 16-bit terms each, every term packed: the first takes the
// leading bits of a value, the next the leading bits of what is left. fp16 cut
// toward zero (one instruction for both values) keeps 11 bits a term, 22 in
// two; bf16 keeps 8 (cut by taking the upper half words), all 24 in three.
template <int TY>
constexpr int TERMS = TY == ATTN_F32 ? 1 : TY == ATTN_F16 ? 2 : 3;
template <int TY>
__device__ __forceinline__ void split(float x, float y, uint32_t (&w)[TERMS<TY>]) {
    if constexpr (TY == ATTN_F16) {
        const auto h = __builtin_amdgcn_cvt_pkrtz(x, y);
        w[0] = bits<uint32_t>(h);
        w[1] = bits<uint32_t>(__builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.0f, x), fmaf((float)h[1], -1.0f, y)));
    } else {
#pragma unroll
        for (int n = 0; n < 3; n++) {
            w[n] = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302u);
            x -= __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
            y -= __uint_as_float(__float_as_uint(y) & 0xFFFF0000u);
        }
    }
}

template <int TY>
__device__ __forceinline__ f32x4 mfma32(const uint4 &a, const uint4 &b, f32x4 c) {
    if constexpr (TY == ATTN_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(bits<f16x8>(a), bits<f16x8>(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(bits<b16x8>(a), bits<b16x8>(b), c, 0, 0, 0);
}

// One value of a cache row as fp32.
template <int TY>
__device__ __forceinline__ float ld_kv(const void *p, uint64_t i) {
    if constexpr (TY == ATTN_F32) return ((const float *)p)[i];
    else if constexpr (TY == ATTN_F16) return (float)((const _Float16 *)p)[i];
    else return __uint_as_float((uint32_t)((const uint16_t *)p)[i] << 16);
}

// How the accumulated product becomes a row's score of a key, in log2 units.
// What a call has of cap and bias is the same for all rows: scalar branches.
struct Score {
    float mul;      // product -> score (with a cap: -> score / cap)
    float cap;      // cap log2(e)
    float slope;    // -slope log2(e)
    float near;     // distance of the row's nearest key
    bool capped, sloped;
    bool bare;      // neither, and a positive factor for every row of the wave
};
struct Row;
__device__ __forceinline__ Score make_score(const AttnArgs &a, const Row &r, float mul);
// scores of the keys j0 + off(r), pos0 = position - j0. The bias counts from the
// row's nearest key on, which the softmax does not notice: a row whose
// document leaves far keys only keeps the bits of its scores.
template <int N, class Off>
__device__ __forceinline__ void scores(const Score &c, float (&y)[N], int32_t pos0, Off off) {
    if (c.capped) {
        // scores well below the cap, as almost all are, need no exponential
        float most = 0.0f;
#pragma unroll
        for (int r = 0; r < N; r++) {
            y[r] *= c.mul;
            most = fmaxf(most, fabsf(y[r]));
        }
        if (__any(most >= 1.0f)) {   // (NaN passes through either way)
#pragma unroll
            for (int r = 0; r < N; r++) {
                y[r] = c.cap * tanh_fast(y[r]);
                __builtin_amdgcn_sched_barrier(0);   // one after another: the rare way takes no registers of the other
            }
        } else {
#pragma unroll
            for (int r = 0; r < N; r++) y[r] = c.cap * tanh_below_1(y[r]);
        }
    } else {
#pragma unroll
        for (int r = 0; r < N; r++) y[r] *= c.mul;
    }
    if (c.sloped) {
        const float p = (float)pos0;
#pragma unroll
        for (int r = 0; r < N; r++) y[r] = fmaf(fabsf(p - (float)off(r)) - c.near, c.slope, y[r]);
    }
}

// What a wave's lane knows about the query row it holds (lanes 16 apart hold
// the same row).
struct Row {
    int32_t row, pos, lo, hi;   // packed row, position, its keys [lo, hi)
    uint32_t head;
    bool valid;
};

__device__ __forceinline__ Row make_row(const AttnArgs &a, uint32_t kvh, uint32_t packed, bool pooled, uint32_t s,
                                        const SeqRows &sr, int32_t n_row) {
    Row r;
    const int32_t t = (int32_t)(packed / a.group);
    r.head = kvh * a.group + packed % a.group;
    r.row = sr.first + t;
    r.valid = t < n_row;
    r.pos = r.lo = r.hi = 0;
    if (r.valid) {
        SeqRows own = sr;
        if (pooled) {
            s = seq_of_row(a, r.row);
            own = seq_rows(a, s);
            r.valid = r.row >= own.first && r.row < own.last && r.row - own.first < (int32_t)a.max_q;
        }
        r.pos = row_pos(a, own, r.row);
        r.hi = (int32_t)a.n_shared + own.len;
        if (a.causal) {
            int32_t upto = r.pos + 1;
            if (a.prefix_len) upto = max(upto, a.prefix_len[s]);
            r.hi = min(r.hi, upto);
        }
        // (kept within the axis, so that no sum of positions leaves 32 bits)
        if (a.doc_start) r.lo = min(max(r.lo, a.doc_start[r.row]), (int32_t)a.n_shared + own.len);
        if (a.doc_end) r.hi = min(r.hi, a.doc_end[r.row]);
        r.hi = max(r.hi, 0);
        if (!r.valid) r.lo = r.hi = 0;
    }
    return r;
}

__device__ __forceinline__ Score make_score(const AttnArgs &a, const Row &r, float mul) {
    Score c;
    c.capped = (__float_as_uint(a.softcap) << 1) != 0;
    c.sloped = a.slopes != nullptr;
    c.cap = a.softcap * LOG2E;
    c.mul = c.capped ? mul / a.softcap : mul * LOG2E;
    c.slope = c.sloped && r.valid ? a.slopes[r.head] * -LOG2E : 0.0f;
    c.near = (float)max(max(r.lo - r.pos, r.pos - r.hi + 1), 0);
    c.bare = !c.capped && !c.sloped && !__any(!(c.mul > 0.0f));
    return c;
}

// min / max over the wave of an integer that 16-lane rows hold alike
__device__ __forceinline__ int32_t row16_min(int32_t v) {
    v = min(v, dpp_i<DPP_XOR1>(v));
    v = min(v, dpp_i<DPP_XOR2>(v));
    v = min(v, dpp_i<DPP_HALF_MIRROR>(v));
    return min(v, dpp_i<DPP_MIRROR>(v));
}

template <int TY, int D>
struct Tile {
    static constexpr int KT = TY == ATTN_F32 ? 16 : 32;          // keys per tile
    static constexpr int DPL = D / 16;                           // columns of V per lane
    static constexpr int EB = TY == ATTN_F32 ? 4 : 2;            // bytes per cache value
    static constexpr int KC = TY == ATTN_F32 ? D / 16 : D / 32;  // 16-byte pieces of a key row per lane
    static constexpr int KR = KT / 16;                           // key rows per lane
    static constexpr int VR = KT / 4;                            // value rows per lane
    static constexpr int VW = DPL * EB / 4;                      // dwords of a value row per lane
};

// The keys and values of one tile in registers. K: lane l holds of key rows
// l % 16 (+ 16) the pieces 8 (l / 16) + 32 c (fp32: 4 (l / 16) + 16 c). V: of
// rows 4 (l / 16) + r (+ 16) the columns DPL (l % 16) ...
template <int TY, int D>
struct Frag {
    using G = Tile<TY, D>;
    static constexpr bool FROM_LDS = false;
    static constexpr int KR = G::KR;
    uint4 k[G::KR][G::KC];
    uint32_t v[G::VR][G::VW];

    // rows j0 ..; rows from `end` on repeat the last one before it: their
    // scores are masked, their values weigh zero and are some row's own
    __device__ __forceinline__ void load_keys(const char *base, uint32_t row_bytes, int32_t j0, int32_t end, int lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        const char *p = base + (uint64_t)(uint32_t)j0 * row_bytes + g * 16;
        const int32_t n = end - j0;
#pragma unroll
        for (int t = 0; t < G::KR; t++) {
            const uint32_t off = (uint32_t)min((int32_t)c + 16 * t, n - 1) * row_bytes;
#pragma unroll
            for (int i = 0; i < G::KC; i++) k[t][i] = *(const uint4 *)(p + off + i * 64);
        }
    }
    __device__ __forceinline__ void load_values(const char *base, uint32_t row_bytes, int32_t j0, int32_t end, int lane) {
        const uint32_t c = lane & 15, g = lane >> 4;
        const char *p = base + (uint64_t)(uint32_t)j0 * row_bytes + c * (G::DPL * G::EB);
        const int32_t n = end - j0;
#pragma unroll
        for (int r = 0; r < G::VR; r++)
            ldv(r, p + (uint32_t)min((int32_t)(4 * g) + (r & 3) + (r >> 2) * 16, n - 1) * row_bytes);
    }
    static constexpr int PLANES = 1;
    __device__ __forceinline__ uint4 key(int t, int i, int) const { return k[t][i]; }
    // V^T's operand for columns DPL (l % 16) + t: halves of 4 + 4 rows exchanged
    __device__ __forceinline__ uint4 value(int t, int) const {
        const uint32_t sel = t & 1 ? 0x07060302u : 0x05040100u;
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = __builtin_amdgcn_perm(v[2 * i + 1][t / 2], v[2 * i][t / 2], sel);
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    __device__ __forceinline__ float value32(int r, int t) const { return __uint_as_float(v[r][t]); }
    __device__ __forceinline__ void ldv(int r, const char *p) {
        if constexpr (G::VW >= 4) {
#pragma unroll
            for (int w = 0; w < G::VW; w += 4) {
                const uint4 x = *(const uint4 *)(p + 4 * w);
                v[r][w] = x.x, v[r][w + 1] = x.y, v[r][w + 2] = x.z, v[r][w + 3] = x.w;
            }
        } else {
            const uint2 x = *(const uint2 *)p;
            v[r][0] = x.x, v[r][1] = x.y;
        }
    }
};

// The query operand of 16 rows: fp32 pieces, or the 16-bit terms of each value,
// in registers or in LDS.
template <int TY, int D>
struct QueryRegs {
    uint4 v[TERMS<TY>][Tile<TY, D>::KC];
    __device__ __forceinline__ uint4 get(int n, int c) const { return v[n][c]; }
    __device__ __forceinline__ void put(int n, int c, const uint4 &x) { v[n][c] = x; }
};
template <int TY, int D>
struct QueryLds {
    static constexpr int BYTES = TERMS<TY> * Tile<TY, D>::KC * 1024;
    char *p;            // the lane's 16 bytes of piece 0
    int first, step;    // pieces that this wave puts there
    __device__ __forceinline__ uint4 get(int n, int c) const {
        return *(const uint4 *)(p + (n * Tile<TY, D>::KC + c) * 1024);
    }
    __device__ __forceinline__ void put(int n, int c, const uint4 &x) const {
        if (c % step == first) *(uint4 *)(p + (n * Tile<TY, D>::KC + c) * 1024) = x;
    }
};

// A wave's running state over its 16 rows.
template <int TY, int D>
struct Wave16 {
    using G = Tile<TY, D>;
    Score sc;
    float m, l;
    f32x4 o[G::DPL];   // o[t][r]: column DPL (4 (l / 16) + r) + t of row l % 16

    template <class Query>
    __device__ __forceinline__ void init(const AttnArgs &a, const Row &r, int lane, Query &q) {
        constexpr int E = TY == ATTN_F32 ? 4 : 8;   // values per piece
        const uint32_t g = lane >> 4;
        const float *qp = a.q + ((uint64_t)(uint32_t)(r.valid ? r.row : 0) * a.n_head + r.head) * D + g * E;
        float v[G::KC][E];
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < G::KC; c++)
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const float4 x = *(const float4 *)(qp + c * (TY == ATTN_F32 ? 16 : 32) + i);
                v[c][i] = x.x, v[c][i + 1] = x.y, v[c][i + 2] = x.z, v[c][i + 3] = x.w;
            }
        float mul = a.scale, up = 1.0f;
        if constexpr (TY == ATTN_F16) {
            // fp16 terms: the row is brought to 2^12 by a power of two, so
            // that neither a large q overflows nor a small one loses bits
#pragma unroll
            for (int c = 0; c < G::KC; c++)
#pragma unroll
                for (int i = 0; i < E; i++) top = fmaxf(top, fabsf(v[c][i]));
            top = rows_max(top);
            int e = (int)((__float_as_uint(top) >> 23) & 255) - 127;
            e = min(max(e, -100), 100);
            up = __uint_as_float((uint32_t)(127 + 12 - e) << 23);
            mul = a.scale * __uint_as_float((uint32_t)(127 - 12 + e) << 23);
        }
#pragma unroll
        for (int c = 0; c < G::KC; c++) {
            if constexpr (TY == ATTN_F32) {
                q.put(0, c, make_uint4(__float_as_uint(v[c][0]), __float_as_uint(v[c][1]), __float_as_uint(v[c][2]),
                                       __float_as_uint(v[c][3])));
            } else {
                uint32_t w[4][TERMS<TY>];
#pragma unroll
                for (int i = 0; i < 4; i++) split<TY>(v[c][2 * i] * up, v[c][2 * i + 1] * up, w[i]);
#pragma unroll
                for (int n = 0; n < TERMS<TY>; n++) q.put(n, c, make_uint4(w[0][n], w[1][n], w[2][n], w[3][n]));
            }
        }
        sc = make_score(a, r, mul);
        m = NEG_INF;
        l = 0.0f;
#pragma unroll
        for (int t = 0; t < G::DPL; t++) o[t] = f32x4{0, 0, 0, 0};
    }

    // The weights of one tile from its products, and the running maximum and sum; keys
    // from `end` on are not of its segment; whole: the row sees all of them.
    template <int VR>
    __device__ __forceinline__ void weights(float (&y)[VR], const Row &row, int32_t j0, int32_t end, bool whole,
                                            int lane) {
        const int32_t g4 = 4 * (lane >> 4);
        // with neither cap nor bias the product's factor goes into the exponent's
        // multiply-add, and y stays the bare product
        float mul = 1.0f;
        if (sc.bare) mul = sc.mul;
        else scores(sc, y, row.pos - j0 - g4, [](int r) { return 16 * (r >> 2) + (r & 3); });
        if (!whole) {
            const int32_t hi = min(row.hi, end);
#pragma unroll
            for (int r = 0; r < VR; r++) {
                const int32_t j = j0 + (r >> 2) * 16 + g4 + (r & 3);
                if (j < row.lo || j >= hi) y[r] = NEG_INF;
            }
        }
        float top = y[0];
#pragma unroll
        for (int r = 1; r < VR; r++) top = fmaxf(top, y[r]);
        top = rows_max(top) * mul;
        // the maximum that scales the sums moves only when it falls behind by
        // 2^8: most tiles then leave the accumulators alone
        if (__any(top > m + 8.0f)) {
            const float mn = fmaxf(m, top);
            const float f0 = m == NEG_INF ? 0.0f : exp2_hw(m - mn);
            m = mn;
            l *= f0;
#pragma unroll
            for (int t = 0; t < G::DPL; t++) o[t] *= f0;
        }
        // fp16 terms of p stand 2^7 higher, so that the second ones stay normal
        const float base = (m == NEG_INF ? 0.0f : m) - (TY == ATTN_F16 ? 7.0f : 0.0f);
#pragma unroll
        for (int r = 0; r < VR; r++) {
            y[r] = exp2_hw(fmaf(y[r], mul, -base));
            l += y[r];
        }
    }

    // Whether an accumulator of the lane's row is not finite.
    __device__ __forceinline__ bool odd() const {
        float z = l * 0.0f;
#pragma unroll
        for (int t = 0; t < G::DPL; t++)
#pragma unroll
            for (int r = 0; r < 4; r++) z = fmaf(o[t][r], 0.0f, z);
        return !(z == 0.0f);
    }
};

// use(i, piece i) for i = 0 .. N-1, each piece asked for A uses ahead: an LDS
// read takes about as long as two pieces' products. r: the pieces 0 .. A-1,
// asked for before.
template <int N, int A, class Load, class Use>
__device__ __forceinline__ void ahead(uint4 (&r)[A + 1], Load load, Use use) {
#pragma unroll
    for (int i = 0; i < N; i++) {
        if (i + A < N) r[(i + A) % (A + 1)] = load(i + A);
        __builtin_amdgcn_sched_barrier(0);
        use(i, r[i % (A + 1)]);
    }
}

// One tile of keys for a wave's B blocks of 16 rows: every operand piece of K
// and V is taken once for all of them. keys_done: called when K's are used up.
template <int TY, int D, int B, class Query, class Src, class Then>
__device__ __forceinline__ void attn_step(Wave16<TY, D> (&st)[B], const Query (&q)[B], Src &f, const Row (&row)[B],
                                          int32_t j0, int32_t end, const bool (&whole)[B], int lane, Then keys_done) {
    using G = Tile<TY, D>;
    constexpr int NT = TERMS<TY>, KR = Src::KR, VR = 4 * KR;
    constexpr int A = TY == ATTN_BF16 && D == 256 ? 1 : 2;   // 1: registers
    constexpr int PL = Src::PLANES;
    float y[B][VR];
    f32x4 s[KR][B];
#pragma unroll
    for (int t = 0; t < KR; t++)
#pragma unroll
        for (int b = 0; b < B; b++) s[t][b] = f32x4{0, 0, 0, 0};
    // piece i: neighbours add to different sums; of a value in terms itself, term
    // p meets the terms 0 .. NT-1-p of the other side: what is left out is below 2^-24
    auto product = [&](int i, const uint4 &k) {
        const int t = i % KR, p = i / KR % PL, c = i / KR / PL;
#pragma unroll
        for (int n = 0; n < NT - p; n++)
#pragma unroll
            for (int b = 0; b < B; b++) {
                if constexpr (TY == ATTN_F32) {
                    const f32x4 kv = bits<f32x4>(k), qv = bits<f32x4>(q[b].get(0, c));
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        s[t][b] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], qv[e], s[t][b], 0, 0, 0);
                } else {
                    s[t][b] = mfma32<TY>(k, q[b].get(n, c), s[t][b]);
                }
            }
    };
    constexpr int NK = KR * PL * G::KC;
    auto key = [&](int i) { return f.key(i % KR, i / KR / PL, i / KR % PL); };
    if constexpr (Src::FROM_LDS && TY != ATTN_F32) {
        uint4 r[A + 1];
#pragma unroll
        for (int i = 0; i < A; i++) r[i] = key(i);
        ahead<NK, A>(r, key, product);
    } else {
#pragma unroll
        for (int i = 0; i < NK; i++) product(i, key(i));
    }
#pragma unroll
    for (int t = 0; t < KR; t++)
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int r = 0; r < 4; r++) y[b][4 * t + r] = s[t][b][r];
    keys_done();
    // the first pieces of V are on their way while the weights are formed
    uint4 pre[A + 1];
    if constexpr (Src::FROM_LDS && TY != ATTN_F32) {
#pragma unroll
        for (int i = 0; i < A; i++) pre[i] = f.value(i / PL, i % PL);
        asm volatile("" ::: "memory");
    }
#pragma unroll
    for (int b = 0; b < B; b++) st[b].weights(y[b], row[b], j0, end, whole[b], lane);
    if constexpr (TY == ATTN_F32) {
#pragma unroll
        for (int r = 0; r < VR; r++)
#pragma unroll
            for (int t = 0; t < G::DPL; t++) {
                const float v = f.value32(r, t);
#pragma unroll
                for (int b = 0; b < B; b++)
                    st[b].o[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, y[b][r], st[b].o[t], 0, 0, 0);
            }
    } else {
        uint32_t pt[B][4][NT];
#pragma unroll
        for (int b = 0; b < B; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) split<TY>(y[b][2 * i], y[b][2 * i + 1], pt[b][i]);
        auto add = [&](int i, const uint4 &vt) {
            const int t = i / PL, p = i % PL;
#pragma unroll
            for (int n = 0; n < NT - p; n++)
#pragma unroll
                for (int b = 0; b < B; b++)
                    st[b].o[t] = mfma32<TY>(vt, make_uint4(pt[b][0][n], pt[b][1][n], pt[b][2][n], pt[b][3][n]), st[b].o[t]);
        };
        if constexpr (Src::FROM_LDS) {
            ahead<G::DPL * PL, A>(pre, [&](int i) { return f.value(i / PL, i % PL); }, add);
        } else {
#pragma unroll
            for (int t = 0; t < G::DPL; t++) add(t, f.value(t, 0));
        }
    }
}

// Keys [c0, c1) of one segment: the shared prefix or a sequence's own cache.
struct Segment {
    const char *k, *v;    // of key c0's axis origin: key j at (j - origin) rows
    int32_t origin, c0, c1;
    uint32_t row_bytes;
};

__device__ __forceinline__ Segment segment(const AttnArgs &a, uint32_t eb, uint32_t kvh, uint32_t s, bool shared,
                                           int32_t c0, int32_t c1) {
    Segment g;
    if (shared) {
        const uint64_t at = (uint64_t)kvh * a.p_head_stride * eb;
        g.k = (const char *)a.pk + at;
        g.v = (const char *)a.pv + at;
        g.row_bytes = (uint32_t)a.p_row_stride * eb;
        g.origin = 0;
        g.c0 = c0;
        g.c1 = min(c1, (int32_t)a.n_shared);
    } else {
        const uint64_t at = ((uint64_t)s * a.seq_stride + (uint64_t)kvh * a.head_stride) * eb;
        g.k = (const char *)a.k + at;
        g.v = (const char *)a.v + at;
        g.row_bytes = (uint32_t)a.row_stride * eb;
        g.origin = (int32_t)a.n_shared;
        g.c0 = max(c0, (int32_t)a.n_shared);
        g.c1 = c1;
    }
    return g;
}

// A row whose accumulators are not finite, again key by key, so that values
// only of its own keys reach it: in a matrix tile a masked key's infinity or
// NaN meets a zero weight and spoils the rows that do not see it. One wave;
// lane l sums columns l, l + 64, ... (out) over the keys of its own tiles.
template <int TY, int D, int W>
__device__ __forceinline__ void row_again(const AttnArgs &a, uint32_t kvh, uint32_t s, const Row &r, int32_t c0,
                                          int32_t c1, int wave, int lane, float (&acc)[D / 64], float &m, float &l) {
    using G = Tile<TY, D>;
    const float *qp = a.q + ((uint64_t)(uint32_t)r.row * a.n_head + r.head) * D;
    const Score sc = make_score(a, r, a.scale);
    m = NEG_INF;
    l = 0.0f;
#pragma unroll
    for (int e = 0; e < D / 64; e++) acc[e] = 0.0f;
    for (int sg = 0; sg < 2; sg++) {
        const Segment g = segment(a, G::EB, kvh, s, sg == 0, c0, c1);
        for (int32_t j0 = g.c0 + wave * G::KT; j0 < g.c1; j0 += W * G::KT)
            for (int32_t j = max(j0, r.lo); j < min(min(j0 + G::KT, g.c1), r.hi); j++) {
                const uint64_t at = (uint64_t)(uint32_t)(j - g.origin) * g.row_bytes;
                float d = 0.0f;
#pragma unroll
                for (int e = 0; e < D / 64; e++)
                    d = fmaf(qp[lane + 64 * e], ld_kv<TY>(g.k + at, lane + 64 * e), d);
                float yj[1] = {group_sum<64>(d)};
                scores(sc, yj, r.pos - j, [](int) { return 0; });
                const float y = yj[0];
                const float mn = y > m ? y : m;
                const float f0 = m == NEG_INF ? 0.0f : exp2_hw(m - mn);
                const float p = exp2_hw(y - (mn == NEG_INF ? 0.0f : mn));
                l = l * f0 + p;
#pragma unroll
                for (int e = 0; e < D / 64; e++) acc[e] = fmaf(p, ld_kv<TY>(g.v + at, lane + 64 * e), acc[e] * f0);
                m = mn;
            }
    }
    if constexpr (TY == ATTN_F16) {   // as the tiles' sums stand
        l *= 128.0f;
#pragma unroll
        for (int e = 0; e < D / 64; e++) acc[e] *= 128.0f;
    }
}

// The item of a workgroup: which rows over which keys, and where the result goes.
struct Item {
    uint32_t kvh, split, tile, seq;
    bool pooled;
};
__device__ __forceinline__ Item make_item(const AttnArgs &a, uint32_t id) {
    Item it;
    it.pooled = id < a.shared_items;   // the longer ones first
    if (!it.pooled) id -= a.shared_items;
    const uint32_t splits = it.pooled ? a.shared_splits : a.own_splits;
    const uint32_t tiles = it.pooled ? a.shared_tiles : a.own_tiles;
    it.kvh = id % a.n_kv;
    id /= a.n_kv;
    it.split = id % splits;
    id /= splits;
    if (it.pooled || a.by_seq) {
        // tiles of the same keys next to each other: the second reads them from the caches
        it.seq = id / tiles;
        it.tile = tiles - 1 - id % tiles;
    } else {
        // later rows see more keys: they start first, in all sequences
        it.seq = id % a.n_seq;
        it.tile = tiles - 1 - id / a.n_seq;
    }
    return it;
}

// A row's result: the output itself, or one of the partial sums that k_attn_join and k_attn_join_few join.
__device__ __forceinline__ uint64_t row_head(const AttnArgs &a, const Row &r) {
    return (uint64_t)(uint32_t)r.row * a.n_head + r.head;
}
__device__ __forceinline__ uint64_t slot_of(const AttnArgs &a, uint64_t rh, const Item &it) {
    return rh * a.slots + (it.pooled ? a.own_splits : 0) + it.split;
}

// The rows an item's packed rows are counted from, and how many there are.
__device__ __forceinline__ int32_t item_rows(const AttnArgs &a, const Item &it, SeqRows &sr) {
    if (it.pooled) {
        sr.first = a.q_start ? min(max(a.q_start[0], 0), (int32_t)a.n_rows) : 0;
        sr.last = a.q_start ? min(max(a.q_start[a.n_seq], sr.first), (int32_t)a.n_rows) : (int32_t)a.n_rows;
        sr.len = 0;
        return sr.last - sr.first;
    }
    sr = seq_rows(a, it.seq);
    return min(sr.last - sr.first, (int32_t)a.max_q);
}

// Of a wave's 16 rows: the keys some row sees among those the item is for,
// [lo, hi), and the keys that every row sees, [all_lo, all_hi).
struct Span {
    int32_t lo, hi, all_lo, all_hi;
};
__device__ __forceinline__ Span wave_span(const AttnArgs &a, const Item &it, const SeqRows &sr, const Row &row) {
    int32_t kb = 0, ke = (int32_t)a.n_shared + sr.len;
    if (it.pooled) ke = (int32_t)a.n_shared;
    else if (a.shared_splits) kb = (int32_t)a.n_shared;
    const int32_t rl = max(row.lo, kb), rh = min(row.hi, ke);
    const bool some = rl < rh;
    Span s;
    s.lo = __builtin_amdgcn_readfirstlane(row16_min(some ? rl : INT32_MAX));
    s.hi = __builtin_amdgcn_readfirstlane(-row16_min(some ? -rh : 0));
    s.all_lo = __builtin_amdgcn_readfirstlane(-row16_min(row.valid ? -row.lo : 0));
    s.all_hi = __builtin_amdgcn_readfirstlane(row16_min(row.valid ? row.hi : INT32_MAX));
    return s;
}

// A split's share [c0, c1) of the keys [lo, hi), in whole tiles of `tile` keys.
__device__ __forceinline__ void split_share(const AttnArgs &a, const Item &it, int32_t lo, int32_t hi, uint32_t tile,
                                            int32_t &c0, int32_t &c1) {
    c0 = c1 = 0;
    if (hi <= lo) return;
    const uint32_t n = (uint32_t)(hi - lo), splits = it.pooled ? a.shared_splits : a.own_splits;
    const uint32_t worth = it.pooled ? a.shared_chunk : a.own_chunk;
    const uint32_t used = min((n + worth - 1) / worth, splits);
    const uint32_t chunk = ((n + used - 1) / used + tile - 1) / tile * tile;
    const uint64_t b = (uint64_t)it.split * chunk;
    if (b < n) {
        c0 = lo + (int32_t)b;
        c1 = lo + (int32_t)min((uint64_t)n, b + chunk);
    }
}

// Rows of the wave that met an infinity or NaN, key by key; buf: D floats of LDS of the wave's own.
template <int TY, int D, int W, int CT>
__device__ __forceinline__ void odd_rows(const AttnArgs &a, const Item &it, const Row &row, int32_t c0, int32_t c1,
                                         int wave, int lane, Wave16<CT, D> &st, float *buf) {
    using G = Tile<TY, D>;
    uint64_t odd = __ballot(row.valid && st.odd());
    odd = (odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xFFFF;
    while (odd) {
        const int i = __builtin_ctzll(odd);
        odd &= odd - 1;
        Row r;
        r.row = __builtin_amdgcn_readlane(row.row, i);
        r.pos = __builtin_amdgcn_readlane(row.pos, i);
        r.lo = __builtin_amdgcn_readlane(row.lo, i);
        r.hi = __builtin_amdgcn_readlane(row.hi, i);
        r.head = (uint32_t)__builtin_amdgcn_readlane((int)row.head, i);
        r.valid = true;
        float acc[D / 64], m, l;
        row_again<TY, D, W>(a, it.kvh, it.seq, r, c0, c1, wave, lane, acc, m, l);
#pragma unroll
        for (int e = 0; e < D / 64; e++) buf[lane + 64 * e] = acc[e];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if ((lane & 15) == i) {
            st.m = m;
            st.l = l;
#pragma unroll
            for (int t = 0; t < G::DPL; t++)
#pragma unroll
                for (int q = 0; q < 4; q++) st.o[t][q] = buf[G::DPL * (4 * (lane >> 4) + q) + t];
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// Few rows: the waves of a workgroup share 16 rows and take every W-th tile of
// the keys, straight from memory into the operands' registers. Bound by
// memory: what counts is how many loads are in flight, so the query operand,
// the same for all waves, lies in LDS, and its registers hold more waves. One
// token over 131072 rows of 8 x 128 fp16: 101 us, 5.3 TB/s; over 300 of fp32,
// 7.2 us, a launch and three dependent loads (eight waves: 8.8 to 11 us, the
// larger join in LDS).
constexpr int ROWS_WAVES = 4;
template <int TY, int D, int W>
struct RowsLds {
    union {
        char q[QueryLds<TY, D>::BYTES];
        float o[W][16][D + 4];
    };
    float m[W][16], l[W][16];
    uint64_t at[16];   // packed row x head of each row, ~0 for none
};
template <int TY, int D, int W>
__device__ __forceinline__ void attn_rows_item(const AttnArgs &a, const Item &it, char *shared) {
    using G = Tile<TY, D>;
    auto &lds = *(RowsLds<TY, D, W> *)shared;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    SeqRows sr;
    const int32_t n_row = item_rows(a, it, sr);
    const Row rows[1] = {make_row(a, it.kvh, it.tile * 16 + (lane & 15), it.pooled, it.seq, sr, n_row)};
    const Row &row = rows[0];
    const Span sp = wave_span(a, it, sr, row);
    int32_t c0, c1;
    split_share(a, it, sp.lo, sp.hi, G::KT, c0, c1);

    // a part without keys leaves word of it, and that is all
    if (c0 >= c1 && a.slots) {
        if (wave == 0 && lane < 16 && row.valid) a.ml[slot_of(a, row_head(a, row), it)] = make_float2(NEG_INF, 0.0f);
        return;
    }

    // the wave's first tile is asked for before q is waited for (with 256-wide
    // heads there are no registers for both)
    Segment g = segment(a, G::EB, it.kvh, it.seq, true, c0, c1);
    int32_t j = g.c0 + wave * G::KT;
    bool own = false;
    if (j >= g.c1) {
        g = segment(a, G::EB, it.kvh, it.seq, false, c0, c1);
        j = g.c0 + wave * G::KT;
        own = true;
    }
    Frag<TY, D> f;
    auto load = [&] {
        f.load_keys(g.k, g.row_bytes, j - g.origin, g.c1 - g.origin, lane);
        f.load_values(g.v, g.row_bytes, j - g.origin, g.c1 - g.origin, lane);
    };
    if (D <= 128 && j < g.c1) load();
    Wave16<TY, D> sts[1], &st = sts[0];
    QueryLds<TY, D> q[1] = {{lds.q + lane * 16, wave, W}};
    st.init(a, row, lane, q[0]);
    __syncthreads();
    if (D > 128 && j < g.c1) load();
    while (j < g.c1) {
        const bool whole[1] = {j >= sp.all_lo && j + G::KT <= min(sp.all_hi, g.c1)};
        const int32_t at = j, end = g.c1;
        j += W * G::KT;
        if (j >= g.c1 && !own) {
            g = segment(a, G::EB, it.kvh, it.seq, false, c0, c1);
            j = g.c0 + wave * G::KT;
            own = true;
        }
        asm volatile("" ::: "memory");   // q's pieces are read again for each tile, not kept
        // the next tile's keys are asked for when these have been used, its values behind them
        attn_step<TY, D, 1>(sts, q, f, rows, at, end, whole, lane, [&] {
            if (j < g.c1) f.load_keys(g.k, g.row_bytes, j - g.origin, g.c1 - g.origin, lane);
            asm volatile("" ::: "memory");
        });
        if (j < g.c1) f.load_values(g.v, g.row_bytes, j - g.origin, g.c1 - g.origin, lane);
    }
    st.l = rows_sum(st.l);
    __syncthreads();   // q is done with: its LDS takes the sums
    odd_rows<TY, D, W>(a, it, row, c0, c1, wave, lane, st, &lds.o[wave][0][0]);

    // the waves' sums of the same rows, joined in LDS
    if (lane < 16) {
        lds.m[wave][lane] = st.m;
        lds.l[wave][lane] = st.l;
        if (wave == 0) lds.at[lane] = row.valid ? row_head(a, row) : ~0ull;
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
#pragma unroll
        for (int t = 0; t < G::DPL; t += 4)
            *(float4 *)&lds.o[wave][lane & 15][G::DPL * (4 * (lane >> 4) + q) + t] =
                make_float4(st.o[t][q], st.o[t + 1][q], st.o[t + 2][q], st.o[t + 3][q]);
    __syncthreads();
    // thread: row tid / (4 W), columns 4 (tid % (4 W)), + 16 W, ...
    const int i = threadIdx.x / (4 * W);
    const uint64_t rh = lds.at[i];
    if (rh == ~0ull) return;
    float m = NEG_INF, l = 0.0f, w[W];
#pragma unroll
    for (int k = 0; k < W; k++) m = fmaxf(m, lds.m[k][i]);
#pragma unroll
    for (int k = 0; k < W; k++) {
        w[k] = lds.l[k][i] == 0.0f ? 0.0f : exp2_hw(lds.m[k][i] - m);
        l += lds.l[k][i] * w[k];
    }
    float *dst;
    float f0 = 1.0f;
    if (a.slots) {
        const uint64_t at = slot_of(a, rh, it);
        if (threadIdx.x % (4 * W) == 0) a.ml[at] = make_float2(m, l);
        if (l == 0.0f) return;
        dst = a.acc + at * D;
    } else {
        f0 = l == 0.0f ? 0.0f : 1.0f / l;
        dst = a.out + rh * D;
    }
#pragma unroll
    for (int c = 0; c < D; c += 16 * W) {
        const int col = c + threadIdx.x % (4 * W) * 4;
        if (col >= D) break;
        float x[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < W; k++) {
            const float4 v = *(const float4 *)&lds.o[k][i][col];
            const float e[4] = {v.x, v.y, v.z, v.w};
            if (w[k] == 0.0f) continue;
#pragma unroll
            for (int n = 0; n < 4; n++) x[n] = fmaf(e[n], w[k], x[n]);
        }
        *(float4 *)(dst + col) = make_float4(x[0] * f0, x[1] * f0, x[2] * f0, x[3] * f0);
    }
}

// Keys and values of NK keys in LDS, for all waves of a workgroup. K row by
// row, 16 bytes of padding each: the 16 rows that a wave's lanes read 16 bytes
// of lie in different banks. 16-bit V in the order of the operand that V^T's
// product takes (column tile, lane, 8 keys): a thread loads 4 rows of 4
// columns and exchanges halves once, where every wave would do it again. fp32
// V row by row.
template <int TY, int D, int NTHREADS>
struct Stage {
    using G = Tile<TY, D>;
    // keys of a stage: few enough for two workgroups on a CU (fp32, 64 wide: four)
    static constexpr int NK = TY == ATTN_F32 ? (D == 256 ? 16 : 32) : D == 256 ? 32 * (NTHREADS / 256) : 64;
    static constexpr int KROW = D * G::EB + 16, VBYTES = TY == ATTN_F32 ? NK * KROW : NK * D * 2;
    static constexpr int BYTES = NK * KROW + VBYTES;
    static constexpr int PER_ROW = D * G::EB / 16;                            // 16-byte pieces of a row
    static constexpr int FK = NK < 32 ? NK : 32;                              // keys of a part
    static constexpr int PARTS = NK / FK;
    static constexpr int SK = FK;                                             // keys worked on at a time
    static constexpr int KN = FK * PER_ROW / NTHREADS;                        // pieces of K per thread
    static constexpr int UNITS = FK / 4 * (D / 4);                            // 4 x 4 blocks of V
    static constexpr int VN = (UNITS + NTHREADS - 1) / NTHREADS;              // blocks per thread
    static_assert(FK * PER_ROW % NTHREADS == 0, "whole pieces per thread");

    u32x4 k[KN];
    uint2 v[TY == ATTN_F32 ? 2 * KN : VN * 4];

    // rows j0 .. j0 + FK from memory; rows from `end` on repeat the last one before it
    __device__ __forceinline__ void fetch(const char *kb, const char *vb, uint32_t row_bytes, int32_t j0, int32_t end) {
        const uint64_t at = (uint64_t)(uint32_t)j0 * row_bytes;
        const char *kp = kb + at, *vp = vb + at;
        const uint32_t last = (uint32_t)min(end - j0, FK) - 1;
#pragma unroll
        for (int n = 0; n < KN; n++) {
            const uint32_t id = threadIdx.x + NTHREADS * n;
            const uint32_t off = min(id / PER_ROW, last) * row_bytes + id % PER_ROW * 16;
            k[n] = *(const u32x4 *)(kp + off);
            if constexpr (TY == ATTN_F32) {
                const uint4 x = *(const uint4 *)(vp + off);
                v[2 * n] = make_uint2(x.x, x.y), v[2 * n + 1] = make_uint2(x.z, x.w);
            }
        }
        if constexpr (TY != ATTN_F32) {
#pragma unroll
            for (int n = 0; n < VN; n++) {
                const uint32_t id = threadIdx.x + NTHREADS * n;
                if (UNITS % NTHREADS == 0 || id < UNITS) {
                    const uint32_t rows = id / (D / 4) * 4, col = id % (D / 4) * 8;
#pragma unroll
                    for (int r = 0; r < 4; r++) v[4 * n + r] = *(const uint2 *)(vp + min(rows + r, last) * row_bytes + col);
                }
            }
        }
    }
    // into part `part` of a stage
    __device__ __forceinline__ void store(char *lds, int part) const {
        char *kl = lds + part * FK * KROW, *vl = lds + NK * KROW + part * (TY == ATTN_F32 ? FK * KROW : FK * D * 2);
#pragma unroll
        for (int n = 0; n < KN; n++) {
            const uint32_t id = threadIdx.x + NTHREADS * n;
            *(u32x4 *)(kl + id / PER_ROW * KROW + id % PER_ROW * 16) = k[n];
            if constexpr (TY == ATTN_F32)
                *(uint4 *)(vl + id / PER_ROW * KROW + id % PER_ROW * 16) =
                    make_uint4(v[2 * n].x, v[2 * n].y, v[2 * n + 1].x, v[2 * n + 1].y);
        }
        if constexpr (TY != ATTN_F32) {
#pragma unroll
            for (int n = 0; n < VN; n++) {
                const uint32_t id = threadIdx.x + NTHREADS * n;
                if (UNITS % NTHREADS == 0 || id < UNITS) {
                    // rows 4 q ..: half q / 4 of the operand's keys, lane row q % 4
                    const uint32_t q = id / (D / 4), col = id % (D / 4) * 4;
                    const uint32_t half = q / 4, lane0 = q % 4 * 16 + col / G::DPL, t0 = col % G::DPL;
                    char *p = vl + (t0 * 64 + lane0) * 16 + half * 8;
                    const uint2 *x = v + 4 * n;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;
                        const uint32_t r0 = e < 2 ? x[0].x : x[0].y, r1 = e < 2 ? x[1].x : x[1].y;
                        const uint32_t r2 = e < 2 ? x[2].x : x[2].y, r3 = e < 2 ? x[3].x : x[3].y;
                        *(uint2 *)(p + e * 1024) =
                            make_uint2(__builtin_amdgcn_perm(r1, r0, sel), __builtin_amdgcn_perm(r3, r2, sel));
                    }
                }
            }
        }
    }
    // the operands of one of its tiles, as Frag gives them
    struct View {
        static constexpr bool FROM_LDS = true;
        static constexpr int KR = SK / 16, PLANES = 1;
        const char *kp, *vp;
        __device__ __forceinline__ uint4 key(int t, int i, int) const { return *(const uint4 *)(kp + t * 16 * KROW + i * 64); }
        __device__ __forceinline__ uint4 value(int t, int) const { return *(const uint4 *)(vp + t * 1024); }
        __device__ __forceinline__ float value32(int r, int t) const { return *(const float *)(vp + ((r >> 2) * 16 + (r & 3)) * KROW + t * 4); }
    };
    static __device__ __forceinline__ View view(const char *lds, int sub, int lane) {
        View w;
        const int c = lane & 15, g = lane >> 4;
        w.kp = lds + (sub * SK + c) * KROW + g * 16;
        if constexpr (TY == ATTN_F32) w.vp = lds + NK * KROW + (sub * SK + 4 * g) * KROW + c * (G::DPL * 4);
        else w.vp = lds + NK * KROW + sub * (32 * D * 2) + lane * 16;
        return w;
    }
};

// fp32 keys and values in LDS as three bf16 terms each (all 24 bits), laid out
// as Stage's 16-bit ones, a plane for each term: six bf16 products for one of
// fp32 take 6/16 of its time on the matrix units.
template <int D, int NTHREADS>
struct StageTerms {
    using G = Tile<ATTN_BF16, D>;
    static constexpr int NK = 32, FK = 32, PARTS = 1, SK = 32;
    static constexpr int KROW = D * 2 + 16, KPLANE = NK * KROW, VPLANE = NK * D * 2;
    static constexpr int BYTES = 3 * (KPLANE + VPLANE);
    static constexpr int PER_ROW = D / 4;                                     // 16-byte pieces of a row
    static constexpr int KN = FK * PER_ROW / NTHREADS;                        // pieces of K per thread
    static constexpr int UNITS = FK / 4 * (D / 4);                            // 4 x 4 blocks of V
    static_assert(FK * PER_ROW % NTHREADS == 0 && UNITS <= NTHREADS, "K in whole pieces, V in one block per thread");

    f32x4 k[KN], v[4];

    __device__ __forceinline__ void fetch(const char *kb, const char *vb, uint32_t row_bytes, int32_t j0, int32_t end) {
        const uint64_t at = (uint64_t)(uint32_t)j0 * row_bytes;
        const char *kp = kb + at, *vp = vb + at;
        const uint32_t last = (uint32_t)min(end - j0, FK) - 1;
#pragma unroll
        for (int n = 0; n < KN; n++) {
            const uint32_t id = threadIdx.x + NTHREADS * n;
            k[n] = *(const f32x4 *)(kp + (min(id / PER_ROW, last) * row_bytes + id % PER_ROW * 16));
        }
        if (threadIdx.x < UNITS) {
            const uint32_t rows = threadIdx.x / (D / 4) * 4, col = threadIdx.x % (D / 4) * 16;
#pragma unroll
            for (int r = 0; r < 4; r++) v[r] = *(const f32x4 *)(vp + (min(rows + r, last) * row_bytes + col));
        }
    }
    __device__ __forceinline__ void store(char *lds, int) const {
#pragma unroll
        for (int n = 0; n < KN; n++) {
            const uint32_t id = threadIdx.x + NTHREADS * n;
            char *p = lds + id / PER_ROW * KROW + id % PER_ROW * 8;
            uint32_t lo[3], hi[3];
            split<ATTN_BF16>(k[n][0], k[n][1], lo);
            split<ATTN_BF16>(k[n][2], k[n][3], hi);
#pragma unroll
            for (int t = 0; t < 3; t++) *(uint2 *)(p + t * KPLANE) = make_uint2(lo[t], hi[t]);
        }
        if (threadIdx.x < UNITS) {
            const uint32_t q = threadIdx.x / (D / 4), col = threadIdx.x % (D / 4) * 4;
            const uint32_t half = q / 4, lane0 = q % 4 * 16 + col / G::DPL, t0 = col % G::DPL;
            char *p = lds + 3 * KPLANE + (t0 * 64 + lane0) * 16 + half * 8;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                uint32_t lo[3], hi[3];
                split<ATTN_BF16>(v[0][e], v[1][e], lo);
                split<ATTN_BF16>(v[2][e], v[3][e], hi);
#pragma unroll
                for (int t = 0; t < 3; t++) *(uint2 *)(p + t * VPLANE + e * 1024) = make_uint2(lo[t], hi[t]);
            }
        }
    }
    struct View {
        static constexpr bool FROM_LDS = true;
        static constexpr int KR = SK / 16, PLANES = 3;
        const char *kp, *vp;
        __device__ __forceinline__ uint4 key(int t, int i, int p) const {
            return *(const uint4 *)(kp + p * KPLANE + t * 16 * KROW + i * 64);
        }
        __device__ __forceinline__ uint4 value(int t, int p) const { return *(const uint4 *)(vp + p * VPLANE + t * 1024); }
    };
    static __device__ __forceinline__ View view(const char *lds, int, int lane) {
        View w;
        w.kp = lds + (lane & 15) * KROW + (lane >> 4) * 16;
        w.vp = lds + 3 * KPLANE + lane * 16;
        return w;
    }
};
// How a tile's keys are staged, and the type its products are formed in.
template <int TY, int D, int NTHREADS>
struct Staging {
    static constexpr int CT = TY;
    using S = Stage<TY, D, NTHREADS>;
};
template <int NTHREADS>
struct Staging<ATTN_F32, 64, NTHREADS> {
    static constexpr int CT = ATTN_BF16;
    using S = StageTerms<64, NTHREADS>;
};
template <int NTHREADS>
struct Staging<ATTN_F32, 128, NTHREADS> {
    static constexpr int CT = ATTN_BF16;
    using S = StageTerms<128, NTHREADS>;
};

// Many rows: the waves of a workgroup, 16 B rows each, walk the same keys,
// staged through LDS for all of them (two buffers: the next keys are on their
// way from memory while these are worked on, one barrier per stage). Bound by
// the matrix units and the weights' arithmetic by turns: 32 heads, 4096 rows
// over 4096 keys of 128, fp16 549 us (1.0 PFLOP/s of products formed, two for
// one), bf16 709 us (1.16 PFLOP/s, three for one), fp32 (16 heads, 2048 rows) 337 us (204
// TFLOP/s; the fp32 instructions 560 us).
template <int TY, int D, int B, int W>
struct TileLds {
    char stage[2][Staging<TY, D, 64 * W>::S::BYTES];
    int32_t span[2][W];
};
template <int TY, int D, int B, int W>
__device__ __forceinline__ void attn_tile_item(const AttnArgs &a, const Item &it, char *shared) {
    using G = Tile<TY, D>;
    using S = typename Staging<TY, D, 64 * W>::S;
    constexpr int CT = Staging<TY, D, 64 * W>::CT;
    constexpr int ROWS = 16 * B * W;
    auto &lds = *(TileLds<TY, D, B, W> *)shared;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    SeqRows sr;
    const int32_t n_row = item_rows(a, it, sr);
    Row row[B];
    Span sp[B];
    int32_t lo = INT32_MAX, hi = 0, c0, c1;
#pragma unroll
    for (int b = 0; b < B; b++) {
        row[b] = make_row(a, it.kvh, it.tile * ROWS + (wave * B + b) * 16 + (lane & 15), it.pooled, it.seq, sr, n_row);
        sp[b] = wave_span(a, it, sr, row[b]);
        lo = min(lo, sp[b].lo);
        hi = max(hi, sp[b].hi);
    }
    const int32_t wave_lo = lo, wave_hi = hi;
    if (lane == 0) {
        lds.span[0][wave] = lo;
        lds.span[1][wave] = hi;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) {
        lo = min(lo, lds.span[0][w]);
        hi = max(hi, lds.span[1][w]);
    }
    lo = __builtin_amdgcn_readfirstlane(lo);
    hi = __builtin_amdgcn_readfirstlane(hi);
    split_share(a, it, lo, hi, S::NK, c0, c1);

    if (c0 >= c1 && a.slots) {   // a part without keys
#pragma unroll
        for (int b = 0; b < B; b++)
            if (lane < 16 && row[b].valid) a.ml[slot_of(a, row_head(a, row[b]), it)] = make_float2(NEG_INF, 0.0f);
        return;
    }
    Wave16<CT, D> st[B];
    QueryRegs<CT, D> q[B];
#pragma unroll
    for (int b = 0; b < B; b++) st[b].init(a, row[b], lane, q[b]);
    S stage;
    if (W == 8 ? wave >= 4 : (blockIdx.x >> 8) & 1) __builtin_amdgcn_s_setprio(1);
    for (int sg = 0; sg < 2; sg++) {
        const Segment g = segment(a, G::EB, it.kvh, it.seq, sg == 0, c0, c1);
        if (g.c0 >= g.c1) continue;
        int at = 0;
        __syncthreads();   // the last segment's readers are done
#pragma unroll 1
        for (int part = 0; part < S::PARTS; part++) {
            if (g.c0 + part * S::FK >= g.c1) break;
            stage.fetch(g.k, g.v, g.row_bytes, g.c0 + part * S::FK - g.origin, g.c1 - g.origin);
            stage.store(lds.stage[0], part);
        }
        __syncthreads();
        for (int32_t j = g.c0; j < g.c1; j += S::NK) {
#pragma unroll 1
            for (int part = 0; part < S::PARTS; part++) {
                // the same part of the next stage is on its way while this one is worked on
                const int32_t jn = j + S::NK + part * S::FK;
                if (jn < g.c1) stage.fetch(g.k, g.v, g.row_bytes, jn - g.origin, g.c1 - g.origin);
                const int32_t js = j + part * S::SK;
                if (js < min(wave_hi, g.c1) && js + S::SK > wave_lo) {
                    bool whole[B];
#pragma unroll
                    for (int b = 0; b < B; b++) whole[b] = js >= sp[b].all_lo && js + S::SK <= min(sp[b].all_hi, g.c1);
                    auto view = S::view(lds.stage[at], part, lane);
                    attn_step<CT, D, B>(st, q, view, row, js, g.c1, whole, lane, [] {});
                }
                if (jn < g.c1) stage.store(lds.stage[at ^ 1], part);
            }
            __syncthreads();
            at ^= 1;
        }
    }
#pragma unroll
    for (int b = 0; b < B; b++) {
        st[b].l = rows_sum(st[b].l);
        // which row and head it was is worked out again: two registers less in the loop
        uint32_t packed = it.tile * ROWS + (wave * B + b) * 16 + (lane & 15);
        asm volatile("" : "+v"(packed));
        row[b].row = sr.first + (int32_t)(packed / a.group);
        row[b].head = it.kvh * a.group + packed % a.group;
        odd_rows<TY, D, 1>(a, it, row[b], c0, c1, 0, lane, st[b], (float *)lds.stage[0] + wave * D);
        if (!row[b].valid) continue;
        float *dst;
        float f0 = 1.0f;
        if (a.slots) {
            const uint64_t at = slot_of(a, row_head(a, row[b]), it);
            if (lane < 16) a.ml[at] = make_float2(st[b].m, st[b].l);
            dst = a.acc + at * D;
            if (st[b].l == 0.0f) continue;
        } else {
            f0 = st[b].l == 0.0f ? 0.0f : 1.0f / st[b].l;
            dst = a.out + row_head(a, row[b]) * D;
        }
#pragma unroll
        for (int q = 0; q < 4; q++)
#pragma unroll
            for (int t = 0; t < G::DPL; t += 4)
                *(float4 *)(dst + G::DPL * (4 * (lane >> 4) + q) + t) = make_float4(
                    st[b].o[t][q] * f0, st[b].o[t + 1][q] * f0, st[b].o[t + 2][q] * f0, st[b].o[t + 3][q] * f0);
    }
}

// The kernels. Mixed: a batch's shared prefix for the rows of all sequences
// together (many rows) beside each sequence's own keys (few rows), in one
// launch: 64 requests over a prefix of 16384 bf16 keys and up to 1024 of their
// own 96 us; with the prefix in tiles of 16 rows too (k_attn for all) 130 us.
template <int TY, int D>
__global__ void __launch_bounds__(64 * ROWS_WAVES, D == 64 ? (TY == ATTN_BF16 ? 3 : 4) : D == 128 ? (TY == ATTN_F32 ? 3 : 2) : TY == ATTN_F32 ? 2 : 1) k_attn(const AttnArgs a) {
    __shared__ __align__(16) char lds[sizeof(RowsLds<TY, D, ROWS_WAVES>)];
    attn_rows_item<TY, D, ROWS_WAVES>(a, make_item(a, blockIdx.x), lds);
}
// (eight waves where four would need more registers to stage the keys than there are)
template <int TY, int D>
constexpr int TILE_WAVES = (TY == ATTN_BF16 && D == 256) || (TY == ATTN_F32 && D == 128) ? 8 : 4;
template <int TY, int D>
__global__ void __launch_bounds__((64 * TILE_WAVES<TY, D>), 2) k_attn_tile(const AttnArgs a) {
    constexpr int W = TILE_WAVES<TY, D>, B = attn_tile_rows(TY, D) / (16 * W);
    __shared__ __align__(16) char lds[sizeof(TileLds<TY, D, B, W>)];
    attn_tile_item<TY, D, B, W>(a, make_item(a, blockIdx.x), lds);
}
template <int TY, int D>
__global__ void __launch_bounds__(64 * ROWS_WAVES, 2) k_attn_mixed(const AttnArgs a) {
    constexpr int W = ROWS_WAVES;
    constexpr size_t R = sizeof(RowsLds<TY, D, W>), T = sizeof(TileLds<TY, D, 1, W>);
    __shared__ __align__(16) char lds[R > T ? R : T];
    const Item it = make_item(a, blockIdx.x);
    if (it.pooled) attn_tile_item<TY, D, 1, W>(a, it, lds);
    else attn_rows_item<TY, D, W>(a, it, lds);
}

// The partial sums of a row, joined. Many slots: a workgroup per (row, head),
// its four waves each every fourth slot, eight slots' loads in flight (64
// slots of 32 rows 4.6 us; one wave a row, one slot after another: 12 us).
template <int D>
__global__ void __launch_bounds__(256) k_attn_join(const AttnArgs a) {
    constexpr int E = D / 64, U = 8, SW = 4;
    __shared__ float part[SW][D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t head = blockIdx.x % a.n_head;
    const uint32_t id = blockIdx.x / a.n_head, seq = id / a.max_q, t = id % a.max_q;
    const SeqRows sr = seq_rows(a, seq);
    if ((int32_t)t >= sr.last - sr.first) return;
    const uint64_t rh = (uint64_t)(uint32_t)(sr.first + (int32_t)t) * a.n_head + head;
    float2 ml = make_float2(NEG_INF, 0.0f);
    if ((uint32_t)lane < a.slots) ml = a.ml[rh * a.slots + lane];
    float m = ml.x;
#pragma unroll
    for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float w = ml.y == 0.0f ? 0.0f : exp2_hw(ml.x - m);
    const float l = group_sum<64>(ml.y * w);
    const float f0 = l == 0.0f ? 0.0f : 1.0f / l;
    float x[E];
#pragma unroll
    for (int e = 0; e < E; e++) x[e] = 0.0f;
    const float *p = a.acc + rh * a.slots * D + lane;
    for (uint32_t k0 = wave; k0 < a.slots; k0 += SW * U) {
        float v[U][E];
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int e = 0; e < E; e++) v[u][e] = p[(uint64_t)min(k0 + SW * u, a.slots - 1) * D + 64 * e];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t k = k0 + SW * u;
            const float wk = k < a.slots ? __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), k & 63)) : 0.0f;
            // a slot that weighs nothing may hold anything
#pragma unroll
            for (int e = 0; e < E; e++) x[e] = wk == 0.0f ? x[e] : fmaf(v[u][e], wk, x[e]);
        }
    }
#pragma unroll
    for (int e = 0; e < E; e++) part[wave][lane + 64 * e] = x[e];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int e = 0; e < E; e++) {
#pragma unroll
        for (int k = 1; k < SW; k++) x[e] += part[k][lane + 64 * e];
        a.out[rh * D + lane + 64 * e] = x[e] * f0;
    }
}

// Up to U slots, four or eight: four values a lane, D / 4 lanes per (row,
// head), each with all slots' maxima and sums, all loads at once: 24 heads of
// 64, 1000 rows, two slots, 5.2 us (a wave for each of the rows, a value a
// lane, 9.6), a launch (2.5) where little is to be joined. Only 300 rows of 32
// heads of 64 with six slots lost by it, 44 us to 47 the whole call.
template <int D, int U>
__global__ void __launch_bounds__(256) k_attn_join_few(const AttnArgs a) {
    constexpr uint32_t L = D / 4;
    const uint32_t at = blockIdx.x * (256 / L) + threadIdx.x / L, i = threadIdx.x % L;
    const uint32_t head = at % a.n_head, id = at / a.n_head, seq = id / a.max_q, t = id % a.max_q;
    if (seq >= a.n_seq) return;
    const SeqRows sr = seq_rows(a, seq);
    if ((int32_t)t >= sr.last - sr.first) return;
    const uint64_t rh = (uint64_t)(uint32_t)(sr.first + (int32_t)t) * a.n_head + head;
    const float2 *q = a.ml + rh * a.slots;
    const float4 *p = (const float4 *)(a.acc + rh * a.slots * D) + i;
    float2 ml[U];
    float4 v[U];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) ml[u] = q[min(u, a.slots - 1)];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) v[u] = p[min(u, a.slots - 1) * L];
    float m = NEG_INF, l = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (uint32_t u = 0; u < U; u++) m = fmaxf(m, ml[u].x);
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
        const float w = u >= a.slots || ml[u].y == 0.0f ? 0.0f : exp2_hw(ml[u].x - m);
        l = fmaf(ml[u].y, w, l);
        const float y[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
        // a slot that weighs nothing may hold anything
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = w == 0.0f ? x[e] : fmaf(y[e], w, x[e]);
    }
    const float f0 = l == 0.0f ? 0.0f : 1.0f / l;
    ((float4 *)(a.out + rh * D))[i] = make_float4(x[0] * f0, x[1] * f0, x[2] * f0, x[3] * f0);
}

template <int TY, int D>
static hipError_t attn_run(const AttnArgs &a, const AttnPlan &p, hipStream_t s) {
    const dim3 rows(64 * ROWS_WAVES), tile(64 * TILE_WAVES<TY, D>);
    if (p.form == ATTN_TILES) {
        hipLaunchKernelGGL((k_attn_tile<TY, D>), dim3(p.own_items), tile, 0, s, a);
    } else if (p.form == ATTN_ROWS) {
        hipLaunchKernelGGL((k_attn<TY, D>), dim3(p.own_items + p.shared_items), rows, 0, s, a);
    } else if constexpr (attn_mixed(TY, D)) {
        hipLaunchKernelGGL((k_attn_mixed<TY, D>), dim3(p.own_items + p.shared_items), rows, 0, s, a);
    } else {
        // no registers (256 wide) or LDS (fp32 in terms, 128 wide) for both in one kernel
        AttnArgs own = a, pooled = a;
        own.shared_items = 0;
        pooled.own_items = 0;
        hipLaunchKernelGGL((k_attn<TY, D>), dim3(p.own_items), rows, 0, s, own);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL((k_attn_tile<TY, D>), dim3(p.shared_items), tile, 0, s, pooled);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || !a.slots) return e;
    // four waves a row where many slots meet
    const uint32_t n = a.n_seq * a.max_q;
    const uint32_t few = (n * a.n_head + 1024 / D - 1) / (1024 / D);
    if (a.slots > 8) hipLaunchKernelGGL((k_attn_join<D>), dim3(n * a.n_head), dim3(256), 0, s, a);
    else if (a.slots > 4) hipLaunchKernelGGL((k_attn_join_few<D, 8>), dim3(few), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_attn_join_few<D, 4>), dim3(few), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_attn(AttnArgs a, uint32_t type, uint32_t head_dim, const AttnPlan &p, void *scratch, hipStream_t s) {
    a.own_tiles = p.own_tiles;
    a.own_splits = p.own_splits;
    a.shared_tiles = p.shared_tiles;
    a.shared_splits = p.shared_splits;
    a.slots = p.slots;
    a.by_seq = p.form != ATTN_TILES;
    a.own_items = p.own_items;
    a.shared_items = p.shared_items;
    a.own_chunk = p.own_chunk;
    a.shared_chunk = p.shared_chunk;
    a.acc = (float *)scratch;
    a.ml = (float2 *)((char *)scratch + (uint64_t)a.n_rows * a.n_head * p.slots * head_dim * 4);
    auto go = [&](auto ty) -> hipError_t {
        constexpr int TY = decltype(ty)::value;
        if (head_dim == 64) return attn_run<TY, 64>(a, p, s);
        if (head_dim == 128) return attn_run<TY, 128>(a, p, s);
        return attn_run<TY, 256>(a, p, s);
    };
    if (type == ATTN_F32) return go(std::integral_constant<int, ATTN_F32>());
    if (type == ATTN_F16) return go(std::integral_constant<int, ATTN_F16>());
    return go(std::integral_constant<int, ATTN_BF16>());
}

}  // namespace kq
