// kq_kv.hip — the step between the q/k/v projections and attention: head
// RMSNorm (optional), rotation by position, and the new k and v rows stored in
// their sequences' caches, in the cache's type.
//
//   y = x / sqrt(mean(x^2) + eps) * w over a head's values (with weights);
//   values i and i + n_rot/2 (or 2i and 2i + 1, interleaved) of the first
//   n_rot turn by the angle pos * base^(-2i / n_rot); v is stored as it is.
//
// One workgroup per packed row. The angles are formed once per row, in
// 64 bits (a far position times a small frequency leaves no bits in 32), as
// turns of which only the fraction matters, and their sine and cosine kept in
// LDS for all heads. One wave per head then: D/64 values per lane, the sum of
// squares across the wave, one store. Every head is read once and written
// once; a single token is a launch's latency.
#include <type_traits>

#include "kq_attn.h"

namespace kq {

constexpr uint32_t KV_THREADS = 512;

template <int TY>
__device__ __forceinline__ void st_kv(void *p, uint64_t i, float x) {
    // a cache value is the fp32 value rounded once, to nearest even
    if constexpr (TY == ATTN_F32) ((float *)p)[i] = x;
    else if constexpr (TY == ATTN_F16) ((_Float16 *)p)[i] = (_Float16)x;
    else ((__bf16 *)p)[i] = (__bf16)x;
}

template <int TY, int D>
__global__ void __launch_bounds__(KV_THREADS) k_kv_append(const AttnArgs a, const RopeArgs r) {
    constexpr int E = D / 64;
    __shared__ float cs[D / 2], sn[D / 2];
    const int lane = threadIdx.x & 63;
    const uint32_t wave = threadIdx.x >> 6;
    const int32_t row = (int32_t)blockIdx.x;
    if (a.q_start && row < a.q_start[0]) return;
    const uint32_t s = seq_of_row(a, row);
    const SeqRows sr = seq_rows(a, s);
    if (row < sr.first || row >= sr.last || row - sr.first >= (int32_t)a.max_q) return;
    const int32_t own = sr.len - (sr.last - row);   // its row in the cache
    const uint32_t half = r.n_rot / 2;
    for (uint32_t i = threadIdx.x; i < half; i += KV_THREADS) {
        const double freq = exp2(-2.0 * (double)i / (double)r.n_rot * r.log2_base);
        double turns = (double)(own + (int64_t)r.pos0) * freq * 0.15915494309189533577;
        turns -= rint(turns);
        float sv, cv;
        sincospif((float)(2.0 * turns), &sv, &cv);
        cs[i] = cv;
        sn[i] = sv;
    }
    __syncthreads();
    const uint32_t heads = a.n_head + 2 * a.n_kv;
    for (uint32_t h = wave; h < heads; h += KV_THREADS / 64) {
        const bool is_q = h < a.n_head, is_k = !is_q && h < a.n_head + a.n_kv;
        const uint32_t kh = is_q ? h : is_k ? h - a.n_head : h - a.n_head - a.n_kv;
        if (!is_q && (own < 0 || own >= (int32_t)a.max_kv)) continue;
        const float *src = is_q ? r.q + ((uint64_t)(uint32_t)row * a.n_head + kh) * D
                                : (is_k ? r.k : r.v) + ((uint64_t)(uint32_t)row * a.n_kv + kh) * D;
        float x[E], y[E];
#pragma unroll
        for (int e = 0; e < E; e++) x[e] = src[lane + 64 * e];
        if (is_q || is_k) {
            // the value each one turns with, and its side of the pair
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t i = lane + 64 * e;
                const uint32_t with = i >= r.n_rot ? i : r.interleaved ? i ^ 1 : i < half ? i + half : i - half;
                y[e] = src[with];
            }
            const float *w = is_q ? r.q_w : r.k_w;
            float inv = 1.0f;
            if (w) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < E; e++) ss = fmaf(x[e], x[e], ss);
                inv = 1.0f / sqrtf(group_sum<64>(ss) / (float)D + r.eps);
            }
#pragma unroll
            for (int e = 0; e < E; e++) {
                const uint32_t i = lane + 64 * e;
                float v = x[e], u = y[e];
                const uint32_t with = i >= r.n_rot ? i : r.interleaved ? i ^ 1 : i < half ? i + half : i - half;
                if (w) {
                    v *= inv * w[i];
                    u *= inv * w[with];
                }
                if (i < r.n_rot) {
                    const uint32_t pair = r.interleaved ? i / 2 : i < half ? i : i - half;
                    const bool first = r.interleaved ? !(i & 1) : i < half;
                    const float c = cs[pair], n = sn[pair];
                    v = first ? v * c - u * n : u * n + v * c;
                }
                x[e] = v;
            }
        }
        if (is_q) {
            float *dst = r.q_out + ((uint64_t)(uint32_t)row * a.n_head + kh) * D;
#pragma unroll
            for (int e = 0; e < E; e++) dst[lane + 64 * e] = x[e];
        } else {
            const uint64_t at = (uint64_t)s * a.seq_stride + (uint64_t)(uint32_t)own * a.row_stride + (uint64_t)kh * a.head_stride;
#pragma unroll
            for (int e = 0; e < E; e++) st_kv<TY>(is_k ? r.k_cache : r.v_cache, at + lane + 64 * e, x[e]);
        }
    }
}

hipError_t launch_kv_append(const AttnArgs &a, const RopeArgs &r, uint32_t type, uint32_t head_dim, hipStream_t s) {
    auto go = [&](auto ty) -> hipError_t {
        constexpr int TY = decltype(ty)::value;
        const dim3 g(a.n_rows), b(KV_THREADS);
        if (head_dim == 64) hipLaunchKernelGGL((k_kv_append<TY, 64>), g, b, 0, s, a, r);
        else if (head_dim == 128) hipLaunchKernelGGL((k_kv_append<TY, 128>), g, b, 0, s, a, r);
        else hipLaunchKernelGGL((k_kv_append<TY, 256>), g, b, 0, s, a, r);
        return hipGetLastError();
    };
    if (type == ATTN_F32) return go(std::integral_constant<int, ATTN_F32>());
    if (type == ATTN_F16) return go(std::integral_constant<int, ATTN_F16>());
    return go(std::integral_constant<int, ATTN_BF16>());
}

}  // namespace kq
