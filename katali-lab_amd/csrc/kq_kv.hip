// kq_kv.hip — the step between the q/k/v projections and attention: head
// RMSNorm (optional), rotation by position, and the new k and v rows stored in
// their sequences' caches, in the cache's type.
//
//   y = x / sqrt(mean(x^2) + eps) * w over a head's values (with weights);
//   values i and i + n_rot/2 (or 2i and 2i + 1, interleaved) of the first
//   n_rot turn by the angle pos * base^(-2i / n_rot); v is stored as it is.
//
// A workgroup takes up to KV_PASSES heads for each of its lane groups of one
// packed row (D/4 lanes hold a head, four values each). It asks for all of
// them first, and forms the row's angles while they come: in 64 bits (a far
// position times a small frequency leaves no bits in 32), as turns of which
// only the fraction matters, sine and cosine kept in LDS for all heads. Every
// head is read once and written once: bound by memory, at a single token by a
// launch's latency. 3600 rows of 16 + 2 + 2 heads of 256, fp16: 42 us from memory
// (3.2 TB/s), 36 us from the cache; one row of 32 + 8 + 8 heads of 128: 4.0 us.
#include <type_traits>

#include "kq_attn.h"

namespace kq {

constexpr uint32_t KV_THREADS = 512;
constexpr int KV_PASSES = 3;

// Four cache values: the fp32 values rounded once, to nearest even.
template <int TY>
__device__ __forceinline__ void st_kv(void *p, uint64_t i, const float (&x)[4]) {
    if constexpr (TY == ATTN_F32) {
        *(float4 *)((float *)p + i) = make_float4(x[0], x[1], x[2], x[3]);
    } else if constexpr (TY == ATTN_F16) {
        typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
        *(f16x4 *)((_Float16 *)p + i) = f16x4{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]};
    } else {
        typedef __bf16 b16x4 __attribute__((ext_vector_type(4)));
        *(b16x4 *)((__bf16 *)p + i) = b16x4{(__bf16)x[0], (__bf16)x[1], (__bf16)x[2], (__bf16)x[3]};
    }
}
__device__ __forceinline__ void ld4f(const float *p, float (&x)[4]) {
    const float4 v = *(const float4 *)p;
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
}

template <int TY, int D>
__global__ void __launch_bounds__(KV_THREADS) k_kv_append(const AttnArgs a, const RopeArgs r, uint32_t parts) {
    constexpr uint32_t LPH = D / 4, PER_PASS = KV_THREADS / LPH;   // lanes per head, heads per pass
    __shared__ float cs[D / 2], sn[D / 2];
    __shared__ __align__(16) float wt[2][D];   // the norms' weights of q and k heads
    const int32_t row = (int32_t)(blockIdx.x / parts);
    const uint32_t first = blockIdx.x % parts * (PER_PASS * KV_PASSES) + threadIdx.x / LPH;
    if (a.q_start && row < a.q_start[0]) return;
    const uint32_t s = seq_of_row(a, row);
    const SeqRows sr = seq_rows(a, s);
    if (row < sr.first || row >= sr.last || row - sr.first >= (int32_t)a.max_q) return;
    const int32_t own = sr.len - (sr.last - row);   // its row in the cache
    const uint32_t half = r.n_rot / 2, heads = a.n_head + 2 * a.n_kv;
    const uint32_t e0 = threadIdx.x % LPH * 4;
    // which values these four turn with
    uint32_t with[4];
#pragma unroll
    for (uint32_t e = 0; e < 4; e++) {
        const uint32_t i = e0 + e;
        with[e] = i >= r.n_rot ? i : r.interleaved ? i ^ 1 : i < half ? i + half : i - half;
    }
    const bool apart = !r.interleaved && r.n_rot, quads = half % 4 == 0;

    auto source = [&](uint32_t h) {
        const uint64_t R = (uint64_t)(uint32_t)row;
        return h < a.n_head ? r.q + (R * a.n_head + h) * D
               : h < a.n_head + a.n_kv ? r.k + (R * a.n_kv + (h - a.n_head)) * D
                                       : r.v + (R * a.n_kv + (h - a.n_head - a.n_kv)) * D;
    };
    float x[KV_PASSES][4];
#pragma unroll
    for (int p = 0; p < KV_PASSES; p++) {
        const uint32_t h = first + PER_PASS * p;
        if (h < heads) ld4f(source(h) + e0, x[p]);
    }
    if (threadIdx.x < D) {
        if (r.q_w) wt[0][threadIdx.x] = r.q_w[threadIdx.x];
        if (r.k_w) wt[1][threadIdx.x] = r.k_w[threadIdx.x];
    }
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
#pragma unroll
    for (int p = 0; p < KV_PASSES; p++) {
        const uint32_t h = first + PER_PASS * p;
        if (h >= heads) continue;
        const bool is_q = h < a.n_head, is_v = h >= a.n_head + a.n_kv;
        if (!is_v) {
            // the other values of the pairs: the neighbours, another lane's four, or (pairs that
            // do not stand apart by whole fours) from memory again, before anything is stored
            float y[4];
            if (!apart) {
                y[0] = x[p][1], y[1] = x[p][0], y[2] = x[p][3], y[3] = x[p][2];
            } else if (quads) {
                const int lane = (int)((threadIdx.x & 63) / LPH * LPH + with[0] / 4);
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = __shfl(x[p][e], lane);
            } else {
#pragma unroll
                for (int e = 0; e < 4; e++) y[e] = source(h)[with[e]];
            }
            if (is_q ? r.q_w : r.k_w) {
                const float *w = wt[is_q ? 0 : 1];
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) ss = fmaf(x[p][e], x[p][e], ss);
                const float inv = 1.0f / sqrtf(group_sum<LPH>(ss) / (float)D + r.eps);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[p][e] *= inv * w[e0 + e];
                    y[e] *= inv * w[with[e]];
                }
            }
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t i = e0 + e;
                if (i >= r.n_rot) continue;
                const uint32_t pair = r.interleaved ? i / 2 : i < half ? i : i - half;
                const bool lead = r.interleaved ? !(i & 1) : i < half;
                const float c = cs[pair], n = sn[pair];
                x[p][e] = lead ? x[p][e] * c - y[e] * n : y[e] * n + x[p][e] * c;
            }
        }
        if (is_q) {
            *(float4 *)(r.q_out + ((uint64_t)(uint32_t)row * a.n_head + h) * D + e0) =
                make_float4(x[p][0], x[p][1], x[p][2], x[p][3]);
        } else if (own >= 0 && own < (int32_t)a.max_kv) {
            const uint32_t kh = is_v ? h - a.n_head - a.n_kv : h - a.n_head;
            st_kv<TY>(is_v ? r.v_cache : r.k_cache,
                      (uint64_t)s * a.seq_stride + (uint64_t)(uint32_t)own * a.row_stride + (uint64_t)kh * a.head_stride + e0,
                      x[p]);
        }
    }
}

hipError_t launch_kv_append(const AttnArgs &a, const RopeArgs &r, uint32_t type, uint32_t head_dim, hipStream_t s) {
    auto go = [&](auto ty) -> hipError_t {
        constexpr int TY = decltype(ty)::value;
        const uint32_t per = KV_THREADS / (head_dim / 4) * KV_PASSES;   // heads of a workgroup
        const uint32_t parts = (a.n_head + 2 * a.n_kv + per - 1) / per;
        const dim3 g(a.n_rows * parts), b(KV_THREADS);
        if (head_dim == 64) hipLaunchKernelGGL((k_kv_append<TY, 64>), g, b, 0, s, a, r, parts);
        else if (head_dim == 128) hipLaunchKernelGGL((k_kv_append<TY, 128>), g, b, 0, s, a, r, parts);
        else hipLaunchKernelGGL((k_kv_append<TY, 256>), g, b, 0, s, a, r, parts);
        return hipGetLastError();
    };
    if (type == ATTN_F32) return go(std::integral_constant<int, ATTN_F32>());
    if (type == ATTN_F16) return go(std::integral_constant<int, ATTN_F16>());
    return go(std::integral_constant<int, ATTN_BF16>());
}

}  // namespace kq
