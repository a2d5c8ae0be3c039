// K8 — appending keys and values to an 8-bit cache with one scale per block of tokens and head.
//
// For every (sequence, block of tokens) that receives rows, each kv head and K or V: a = largest magnitude of the new rows,
// s = scale(a), joined with the old scale when the block held tokens already, code = x / s rounded once. The bound is memory:
// 2 bytes read and 1 written per value of a prompt in 16 bits (3 bytes x 2 x Hkv x D per token); a single token per sequence is
// latency. One CTA does one block of one head, so that the rows are read once: each thread keeps its 64 values
// (loaded together) between the maximum and the quotients, and no second pass or second kernel is needed. 64 registers a
// thread keep 1024 threads with 128 bytes each on their way per SM: 43 k tokens of 8 heads x 128 (K and V, bf16 to e4m3, blocks
// of 128) in 49 to 52 us back to back, 5.4 to 5.1 TB/s; with 84 registers 67 us. 32 single tokens 2.9 to 3.1 us in a graph.
// The bound of 64 registers is made for 16-bit rows, which take 32 of them (40 to 56 bytes of spills a thread). Rows in fp32 take all
// 64, so that a part of them goes through local memory (440 bytes of spills a thread for int8, 532 for e4m3): 40 k tokens of 8
// heads x 128 in blocks of 128 take 99 us (e4m3) and 107 us (int8), 4.1 and 3.8 TB/s, where bf16 rows take 44 and 50 us (5.5, 4.9).
//
// The scale of e4m3 codes is a power of two: the format carries its own exponent, so a finer scale would not make a code more
// precise, and multiplying by 2^-e is exact — the code is the value rounded once. int8 codes take a / 127, which spreads the
// block's range over all 255 codes.
#include "common.cuh"
#include "kv_q8.cuh"

namespace {

    constexpr int kVec = 8; // 8-value vectors per thread: block * D = 64 * threads

    struct AppendParams {
        const void    *X[2];     // K, V
        uint8_t       *codes[2]; // [B,Hkv,Lmax,D]
        float         *scales[2];
        int64_t        xs[2][2]; // element strides {token, head}
        int64_t        B, Hkv, Lmax, total;
        int            D, block, vshift, bshift; // D = 8 << vshift, block = 1 << bshift
        const int32_t *cu, *kv_len;
        int            vec_ok; // bases and strides of K and V allow 16-byte loads
    };

    // Eight values as fp32, from one 16-byte vector of a 16-bit type or two of fp32. (Plain loads: the read-only path is for memory that
    // nobody writes while the kernel runs, and the kernel before this one may still be writing the rows when this one starts.)
    template <typename T> struct Row8 {
        uint4 v[sizeof(T) == 4 ? 2 : 1];
        __device__ __forceinline__ void load(const T *p, bool vec_ok) {
            if (vec_ok) {
#pragma unroll
                for (int i = 0; i < (int) (sizeof(v) / 16); ++i) v[i] = reinterpret_cast<const uint4 *>(p)[i];
            } else {
                T *e = reinterpret_cast<T *>(v);
#pragma unroll
                for (int i = 0; i < 8; ++i) e[i] = p[i];
            }
        }
        __device__ __forceinline__ void zero() {
#pragma unroll
            for (int i = 0; i < (int) (sizeof(v) / 16); ++i) v[i] = make_uint4(0, 0, 0, 0);
        }
        // The larger of `m` and the magnitudes, as ordered bits: for the 16-bit types two at a time, in the two halves of m.
        __device__ __forceinline__ uint32_t top(uint32_t m) const {
            const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
            for (int i = 0; i < (int) (sizeof(v) / 4); ++i) {
                if (sizeof(T) == 4) m = m > (w[i] & 0x7fffffffu) ? m : w[i] & 0x7fffffffu;
                else m = __vmaxu2(m, w[i] & 0x7fff7fffu);
            }
            return m;
        }
        // ... and its fp32 bits.
        static __device__ __forceinline__ uint32_t top_bits(uint32_t m) {
            if (sizeof(T) == 4) return m;
            const uint32_t h = m >> 16 > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
            if (std::is_same<T, __nv_bfloat16>::value) return h << 16;
            return __float_as_uint(__half2float(__ushort_as_half((unsigned short) h)));
        }
        __device__ __forceinline__ float get(int i) const { return St<T>::ld(reinterpret_cast<const T *>(v) + i); }
    };

    template <typename T, bool kE4m3> __global__ void __launch_bounds__(512, 2) kv_append_kernel(const AppendParams p) {
        const int     tid = threadIdx.x, nt = blockDim.x, which = blockIdx.z, hk = blockIdx.y;
        const int     D = p.D, block = p.block, sh = p.vshift; // 1 << sh vectors per row
        vkc_grid_dep_wait();
        vkc_grid_dep_launch();
        // the (sequence, block) of this CTA
        int64_t b, x0, n, blk;
        int     start = 0; // tokens the sequence holds
        if (p.cu) {
            int64_t first, x1;
            b   = vkc_packed_find_warp(p.cu, p.kv_len, p.B, p.total, blockIdx.x, p.bshift, 2, &first, &x0, &x1, &start);
            n   = x1 - x0;
            blk = blockIdx.x - first;
        } else {
            b = blockIdx.x, x0 = b, n = 1, blk = 0;
            if (p.kv_len) start = p.kv_len[b];
        }
        if (blk < 0 || start < 0 || start >= p.Lmax) return;
        blk += start >> p.bshift;
        const int64_t lo   = blk << p.bshift;
        const int64_t from = start > lo ? start : lo; // new rows of this block: positions [from, to)
        int64_t       to   = start + n < lo + block ? start + n : lo + block;
        if (to > p.Lmax) to = p.Lmax;
        if (from >= to) return;
        const int  r0 = (int) (from - lo), r1 = (int) (to - lo); // ... as rows of the block
        const bool held = r0 > 0;                                // tokens were there before

        const int64_t row0  = (b * p.Hkv + hk) * p.Lmax + lo;
        uint8_t      *codes = p.codes[which] + row0 * D;
        float        *scale = p.scales[which] + (b * p.Hkv + hk) * (p.Lmax >> p.bshift) + blk;
        const T      *x     = (const T *) p.X[which] + (x0 + from - start) * p.xs[which][0] + hk * p.xs[which][1];
        const float   s_old = held ? *scale : 0.f;

        // vector i of this thread: row first + i * step of the block, always the same dims
        const int     first = tid >> sh, step = block >> 3;
        const int64_t leap = step * p.xs[which][0];
        x += (int64_t) (first - r0) * p.xs[which][0] + (tid - (first << sh)) * 8;
        uint2   *at = reinterpret_cast<uint2 *>(codes) + tid;
        Row8<T>  rows[kVec];
        uint32_t top = 0; // bits of |x| order like the values, infinities and NaN above all
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int r = first + i * step;
            if (r >= r0 && r < r1) rows[i].load(x, p.vec_ok);
            else rows[i].zero();
            x += leap;
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) top = rows[i].top(top);
        top = Row8<T>::top_bits(top);
        __shared__ uint32_t part[16];
        top = __reduce_max_sync(0xffffffffu, top);
        if ((tid & 31) == 0) part[tid >> 5] = top;
        __syncthreads();
        for (int w = 0; w < (nt >> 5); ++w) top = part[w] > top ? part[w] : top;

        const float s_new = q8::scale_of<kE4m3>(top);
        float       s     = s_new;
        if (held) s = (s_new != s_new || s_old != s_old) ? q8::nan_value() : fmaxf(s_new, s_old);
        if (tid == 0) *scale = s; // (read by every thread before the barrier above)
        const q8::Quant<kE4m3> quant(s);
        if (held && s > s_old) { // the older codes, in steps of the larger scale
            const q8::Requant<kE4m3> re(s_old, s);
#pragma unroll
            for (int i = 0; i < kVec; ++i) {
                if (first + i * step < r0) {
                    uint2 c = at[i * nt];
                    c.x = re.four(c.x), c.y = re.four(c.y);
                    at[i * nt] = c;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < kVec; ++i) {
            const int r = first + i * step;
            if (r >= r0 && r < r1) {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = rows[i].get(e);
                at[i * nt] = quant.eight(f);
            }
        }
    }

    template <typename T> void launch_append(vkc_ctx *ctx, bool e4m3, dim3 grid, int threads, cudaStream_t st, const AppendParams &p) {
        if (e4m3) vkc_launch(ctx, kv_append_kernel<T, true>, grid, dim3(threads), 0, st, p);
        else vkc_launch(ctx, kv_append_kernel<T, false>, grid, dim3(threads), 0, st, p);
    }

} // namespace

extern "C" int vkc_kv_append_q8(vkc_ctx *ctx, const vkc_kv_append_q8_args *args, vkc_stream stream) {
    if (!ctx) return VKC_ERR_INVALID;
    VKC_REQUIRE(ctx, args, "kv_append_q8: null arguments");
    const auto [K, V, Kc, Vc, k_scale, v_scale, B, Hkv, Lmax, D, block, total, cu, kv_len, k_strides, v_strides, dtype, cache_dtype] = *args;
    VKC_REQUIRE(ctx, B >= 0 && Hkv >= 1 && Lmax >= 1 && D >= 1 && total >= 0, "kv_append_q8: bad extents");
    VKC_REQUIRE(ctx, dtype == VKC_F32 || dtype == VKC_F16 || dtype == VKC_BF16, "kv_append_q8: bad dtype %d", dtype);
    if (int rc = vkc_q8_check(ctx, "kv_append_q8", B, Hkv, Lmax, D, block, cache_dtype)) return rc;
    VKC_REQUIRE(ctx, total <= INT32_MAX - 1024, "kv_append_q8: more rows than 32-bit offsets reach");
    VKC_REQUIRE(ctx, cu || total == B, "kv_append_q8: without cu every sequence brings one row (total=%lld, B=%lld)", (long long) total, (long long) B);
    if (B == 0 || total == 0) return VKC_OK;
    VKC_REQUIRE(ctx, K && V && Kc && Vc && k_scale && v_scale, "kv_append_q8: null tensor");
    VKC_REQUIRE(ctx, !(((uintptr_t) Kc | (uintptr_t) Vc) & 15), "kv_append_q8: the cache must be 16-byte aligned");
    VKC_REQUIRE(ctx, !(((uintptr_t) K | (uintptr_t) V) & (vkc_dtype_size(dtype) - 1)), "kv_append_q8: K/V are not aligned to their type");
    VKC_REQUIRE(ctx, !(((uintptr_t) k_scale | (uintptr_t) v_scale | (uintptr_t) cu | (uintptr_t) kv_len) & 3), "kv_append_q8: scales, offsets or lengths are not aligned to their type");
    VkcDeviceGuard guard(ctx);
    AppendParams   p;
    p.X[0] = K, p.X[1] = V;
    p.codes[0] = (uint8_t *) Kc, p.codes[1] = (uint8_t *) Vc;
    p.scales[0] = k_scale, p.scales[1] = v_scale;
    const int64_t dense[2] = {Hkv * D, D}, *str[2] = {k_strides[0] || k_strides[1] ? k_strides : dense, v_strides[0] || v_strides[1] ? v_strides : dense};
    const int64_t per16    = 16 / (int64_t) vkc_dtype_size(dtype);
    p.vec_ok               = !(((uintptr_t) K | (uintptr_t) V) & 15);
    for (int w = 0; w < 2; ++w)
        for (int i = 0; i < 2; ++i) {
            p.xs[w][i] = str[w][i];
            if (str[w][i] % per16) p.vec_ok = 0;
        }
    p.B = B, p.Hkv = Hkv, p.Lmax = Lmax, p.total = total, p.D = (int) D, p.vshift = D == 64 ? 3 : D == 128 ? 4 : 5, p.block = (int) block, p.bshift = block == 32 ? 5 : block == 64 ? 6 : 7, p.cu = cu, p.kv_len = kv_len;
    const dim3 grid((unsigned) (cu ? total / block + 2 * B : B), (unsigned) Hkv, 2);
    const int  threads = (int) (block * D / 64);
    const bool e4m3    = cache_dtype == VKC_E4M3;
    cudaStream_t st    = vkc_pick_stream(ctx, stream);
    switch (dtype) {
        case VKC_F32: launch_append<float>(ctx, e4m3, grid, threads, st, p); break;
        case VKC_F16: launch_append<__half>(ctx, e4m3, grid, threads, st, p); break;
        default: launch_append<__nv_bfloat16>(ctx, e4m3, grid, threads, st, p); break;
    }
    return vkc_post_launch(ctx, "kv_append_q8");
}
