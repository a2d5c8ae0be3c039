// K9 — single-query attention over the 8-bit cache (kv_q8.cuh): scores and sums in fp32, each block's scale applied to the
// score (K) and to the probability (V).
#include "kv_q8.cuh"

namespace {

    struct DecQ8Params {
        const void    *Q;
        const uint8_t *Kc, *Vc;
        const float   *ks, *vs;
        void          *O;
        int64_t        Hq, Hkv, Lmax;
        int            block;
        const int32_t *kv_len;
        float          scale_log2;
    };

    __device__ __forceinline__ int64_t q8_len(const DecQ8Params &p, int64_t b) {
        const int64_t len = p.kv_len ? (int64_t) p.kv_len[b] : p.Lmax;
        return len < 0 ? 0 : (len > p.Lmax ? p.Lmax : len);
    }
    template <bool kE4m3> __device__ __forceinline__ float q8_value(uint32_t c) { return kE4m3 ? q8::e4m3_value(c) : (float) (int8_t) c; }

    constexpr int kSimtWarps = 8;

    // SIMT form: one CTA per (query head, sequence), the warps take keys round-robin, a lane holds D / 32 dims of the row.
    template <typename T, int D, bool kE4m3> __global__ void __launch_bounds__(kSimtWarps * 32) attn_decode_q8_simt_kernel(const DecQ8Params p) {
        constexpr int DL = D / 32;
        const int     warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        const int64_t h = blockIdx.x, b = blockIdx.y, hk = h / (p.Hq / p.Hkv), nb = p.Lmax / p.block;
        vkc_grid_dep_wait();
        vkc_grid_dep_launch();
        const int64_t  len = q8_len(p, b);
        const uint8_t *kb = p.Kc + (b * p.Hkv + hk) * p.Lmax * D, *vb = p.Vc + (b * p.Hkv + hk) * p.Lmax * D;
        const float   *ks = p.ks + (b * p.Hkv + hk) * nb, *vs = p.vs + (b * p.Hkv + hk) * nb;
        const T       *q  = (const T *) p.Q + (b * p.Hq + h) * D;
        float          qf[DL], o[DL], m = -INFINITY, l = 0.f;
#pragma unroll
        for (int e = 0; e < DL; ++e) qf[e] = St<T>::ld(q + lane * DL + e) * p.scale_log2, o[e] = 0.f;
        for (int64_t j = warp; j < len; j += kSimtWarps) {
            float s = 0.f;
#pragma unroll
            for (int e = 0; e < DL; ++e) s = fmaf(qf[e], q8_value<kE4m3>(kb[j * D + lane * DL + e]), s);
#pragma unroll
            for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
            s *= ks[j / p.block];
            const float mn = fmaxf(m, s), a = exp2f(m - mn), e1 = exp2f(s - mn), pv = e1 * vs[j / p.block];
            l = l * a + e1;
            m = mn;
#pragma unroll
            for (int e = 0; e < DL; ++e) o[e] = fmaf(pv, q8_value<kE4m3>(vb[j * D + lane * DL + e]), o[e] * a);
        }
        __shared__ float sm[kSimtWarps], sl[kSimtWarps], so[kSimtWarps][D];
        if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
        for (int e = 0; e < DL; ++e) so[warp][lane * DL + e] = o[e];
        __syncthreads();
        for (int d = threadIdx.x; d < D; d += kSimtWarps * 32) {
            float mt = -INFINITY, lt = 0.f, ot = 0.f;
#pragma unroll
            for (int w = 0; w < kSimtWarps; ++w) mt = fmaxf(mt, sm[w]);
#pragma unroll
            for (int w = 0; w < kSimtWarps; ++w) {
                const float a = sm[w] == -INFINITY && sl[w] == 0.f ? 0.f : exp2f(sm[w] - mt);
                lt += sl[w] * a, ot += so[w][d] * a;
            }
            St<T>::st((T *) p.O + (b * p.Hq + h) * D + d, ot / lt); // no key: 0 / 0 = NaN
        }
    }

    template <typename T, int D> void launch_simt(vkc_ctx *ctx, bool e4m3, dim3 grid, cudaStream_t st, const DecQ8Params &p) {
        if (e4m3) vkc_launch(ctx, attn_decode_q8_simt_kernel<T, D, true>, grid, dim3(kSimtWarps * 32), 0, st, p);
        else vkc_launch(ctx, attn_decode_q8_simt_kernel<T, D, false>, grid, dim3(kSimtWarps * 32), 0, st, p);
    }

} // namespace

extern "C" size_t vkc_attn_decode_q8_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lmax, int64_t D) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Lmax <= 0 || D <= 0) return 0;
    return 16;
}

extern "C" int vkc_attn_decode_q8(vkc_ctx *ctx, const void *Q, const void *Kc, const void *Vc, const float *k_scale, const float *v_scale, void *O,
                                  int64_t B, int64_t Hq, int64_t Hkv, int64_t Lmax, int64_t D, int64_t block, const int32_t *kv_len, float scale,
                                  void *workspace, size_t workspace_bytes, int dtype, int cache_dtype, vkc_stream stream) {
    if (!ctx) return VKC_ERR_INVALID;
    VKC_REQUIRE(ctx, B >= 0 && Hq >= 1 && Hkv >= 1 && Lmax >= 1 && D >= 1, "attn_decode_q8: bad extents");
    VKC_REQUIRE(ctx, Hq % Hkv == 0, "attn_decode_q8: Hq=%lld is not a multiple of Hkv=%lld", (long long) Hq, (long long) Hkv);
    if (dtype != VKC_F16 && dtype != VKC_BF16) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "attn_decode_q8: Q and O must be f16 or bf16");
    if (int rc = vkc_q8_check(ctx, "attn_decode_q8", B, Hkv, Lmax, D, block, cache_dtype)) return rc;
    VKC_REQUIRE(ctx, Hq <= 65535 * 16, "attn_decode_q8: extents too large");
    if (B == 0) return VKC_OK;
    VKC_REQUIRE(ctx, Q && Kc && Vc && k_scale && v_scale && O, "attn_decode_q8: null tensor");
    VKC_REQUIRE(ctx, !(((uintptr_t) Q | (uintptr_t) Kc | (uintptr_t) Vc) & 15), "attn_decode_q8: Q and the cache must be 16-byte aligned");
    const size_t need = vkc_attn_decode_q8_workspace_bytes(B, Hq, Hkv, Lmax, D);
    VKC_REQUIRE(ctx, !workspace || (workspace_bytes >= need && !((uintptr_t) workspace & 15)),
                "attn_decode_q8: workspace of %zu bytes is smaller than the %zu required, or not 16-byte aligned", workspace_bytes, need);
    if (ctx->impl == VKC_IMPL_TCGEN05) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "attn_decode_q8: no tensor-core kernel");
    VkcDeviceGuard guard(ctx);
    cudaStream_t   st = vkc_pick_stream(ctx, stream);
    DecQ8Params    p;
    p.Q = Q, p.Kc = (const uint8_t *) Kc, p.Vc = (const uint8_t *) Vc, p.ks = k_scale, p.vs = v_scale, p.O = O;
    p.Hq = Hq, p.Hkv = Hkv, p.Lmax = Lmax, p.block = (int) block, p.kv_len = kv_len;
    p.scale_log2 = scale * 1.4426950408889634f;
    const dim3 grid((unsigned) Hq, (unsigned) B);
    const bool e4m3 = cache_dtype == VKC_E4M3;
#define VKC_Q8_SIMT(T)                                              \
    switch (D) {                                                    \
        case 64: launch_simt<T, 64>(ctx, e4m3, grid, st, p); break;   \
        case 128: launch_simt<T, 128>(ctx, e4m3, grid, st, p); break; \
        default: launch_simt<T, 256>(ctx, e4m3, grid, st, p); break;  \
    }
    if (dtype == VKC_F16) VKC_Q8_SIMT(__half) else VKC_Q8_SIMT(__nv_bfloat16)
#undef VKC_Q8_SIMT
    return vkc_post_launch(ctx, "attn_decode_q8");
}
