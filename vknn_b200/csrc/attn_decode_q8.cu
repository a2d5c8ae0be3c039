// K9 — single-query attention over the 8-bit cache (kv_q8.cuh), bound by the bytes of the cache: 2 * Hkv * len * D per
// sequence and the scales (8 / (block * D) of that). All arithmetic on the sums is fp32; each block's scale multiplies the
// score (K) and the tile's product (V), never a 16-bit operand.
//
// Streaming form. The cache is cut into tiles of 32 keys; the tiles of all (sequence, kv head) units lie on one line and every
// WARP takes an equal run of it, so that the lengths of the sequences do not matter. Each warp has a ring of shared-memory
// stages of its own that its lane 0 fills with two bulk-tensor copies per tile (K, V; 128-byte swizzle), across the ends of
// units: no warp ever waits for another one, and 192 KB are on the way to every SM. (Runs per CTA whose tiles the warps took in
// turn cost three barriers and a merge in shared memory per unit, some 6000 cycles: 64 short sequences took 49 us, not 28.) A tile is
// consumed by warp-level 16x8x16 matrix instructions straight from 8-bit codes:
//   S[heads, 8 keys] += Q[heads, 16 dims] . K^T      B fragments: 4 code bytes of a key -> two f16 pairs
//   O^T[16 dims, heads] += V^T[16 dims, 16 keys] . P^T  A fragments: the bytes of two keys interleaved -> f16 pairs
// The fragment layouts leave two freedoms that make this cheap. The dims of a dot product may be taken in any order as long as Q
// is laid out the same way, so a thread reads whole 16-byte chunks of a key and uses them 4 bytes at a time; and the rows of
// O^T may be any dims, so a thread reads 16 consecutive bytes of each of its keys. The accumulator of S is already the B
// fragment of the second product. e4m3 and int8 codes are exact in f16, and so is Q (bf16 rows are scaled by a power of two
// first), so the products are those of the values; P is rounded to f16 (11 bits, also for bf16 outputs), times 2^7 so that
// probabilities down to 2^-21 of the largest keep all of them.
// Why not tcgen05: at the memory's rate an SM has to convert and multiply 23 codes per clock. The warp-level instructions use 0.42
// of the issue slots and 0.29 of their own pipe for that (profiles) and keep scores and probabilities in registers, where
// the tensor-memory route would carry every tile through it twice; the tensor rate is of no concern at 8 or 16 columns.
// Measured: 32 sequences of 1024 to 8192 tokens, 32/8 heads x 128, 339 MB of e4m3: 64 us with the join, 5.8 TB/s while
// streaming (0.89 of the copy rate); two sequences of up to 131000 tokens, 509 MB: 88 us. Such a batch of 154000 tokens in all,
// 8 kv heads, us and TB/s with the join, groups of 1, 8 and 16 query heads, e4m3: D = 64 (157 MB) 40 / 41 / 49 (3.9, 3.8, 3.2),
// D = 128 59 / 62 / 76 (5.3, 5.1, 4.2), D = 256 103 / 107 / 194 (6.1, 5.9, 3.2). Groups of 9 to 16 keep two sets of Q fragments
// and accumulators in registers and spill 80 to 92 bytes a thread at D = 128 and 420 to 452 at D = 256.
// A unit that lies in one run is finished there; one that is cut leaves a partial (maximum, sum, O) per run in the workspace
// (slot 0: the unit began in an earlier run, slot 1: in this one) and a second kernel joins them in the order of the runs.
// (Joined by the warp whose partial arrives last instead, the batch took 73 us, not 67: the fences hold up the stream.)
// Short caches take one CTA per unit instead (kUnit, one_cta_per_unit): its warps share the unit's tiles, merge once in shared
// memory and store O; one kernel and no workspace.
#include "kv_q8.cuh"
#include "ptx.cuh"
#include "tensormap.cuh"

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

    // SIMT form: one CTA per (query head, sequence), the warps take keys round-robin, a lane holds D / 32 dims of the row. It is the
    // form of groups of more than 16 query heads, which the streaming form's fragments do not hold, and reads the cache once per head,
    // a byte at a time, with no cut along the keys: 32 heads on one kv head, D = 128, 32 sequences of 1024 to 8192 tokens 848 us, one
    // of 131072 tokens 8.7 ms (16 heads in the streaming form: 34 us).
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

    // ---------------------------------------------------------------------------------------------------------------------
    constexpr int kTile     = 32;   // keys per tile
    constexpr int kMaxCtas  = 160;
    constexpr int kMinTiles = 2;    // tiles of a run, at least
    constexpr int kSliceB   = 1024; // sequences per launch (prefix table in shared memory)

    struct StreamParams {
        DecQ8Params q;
        int         B, G; // sequences of this launch, query heads per kv head
        int         runs; // partial slots of the workspace hold this many runs
        bool        unit; // one CTA per unit
        int         block_log2;
        float      *part_o;  // [runs][2][G][D]
        float      *part_ml; // [runs][2][G][2]
        int        *line;    // [B + 1] first line position of each sequence, then the tiles of a run: written for the join
        int        *dev_err;
    };

    // NT = groups of eight query heads. W warps, S ring stages each.
    template <int D, int NT> struct Stream {
        static constexpr int      W = D == 256 ? 4 : 8;
        static constexpr int      S = D == 64 ? 6 : 3;
        static constexpr int      CH = D / 64;   // 16-byte chunks of a key row per thread (QK)
        static constexpr int      MT = D / 16;   // 16-dim row tiles of O^T
        static constexpr uint32_t TILE  = kTile * D; // bytes of a K or V tile
        static constexpr uint32_t oRing = 0;
        static constexpr uint32_t oBar  = oRing + W * S * 2 * TILE;
        static constexpr uint32_t oSc   = oBar + W * S * 8;                      // [W][S][2]
        static constexpr uint32_t oCtl  = oSc + W * S * 8;                       // abort flag
        static constexpr uint32_t oTab  = oCtl + 16;                             // first line position of each sequence
        static constexpr uint32_t total = oTab + (kSliceB + 1) * 4 + 1024;
        static_assert(total <= 227 * 1024, "shared memory budget");
        static_assert(W * NT * 8 * (D + 2) * 4 <= (int) oBar, "the warps' partials fit into the ring");
    };

    // D[16x8] += A[16x16] * B[16x8], f16 operands, fp32 accumulator
    __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    // ... D = A * B, with no accumulator to clear first
    __device__ __forceinline__ void mma16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    }
    // four codes -> two f16 pairs, low pair first
    template <bool kE4m3> __device__ __forceinline__ void codes_to_f16(uint32_t x, uint32_t &lo, uint32_t &hi) {
        if (kE4m3) {
            asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(x));
        } else {
            // code + 128 as the low byte of 0x6400 is 1024 + 128 + code in f16; subtracting 1152 is exact
            const uint32_t  u = x ^ 0x80808080u;
            const uint32_t  l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
            const __half2   off = __half2half2(__ushort_as_half((unsigned short) 0x6480));
            const __half2   a = __hsub2(*reinterpret_cast<const __half2 *>(&l), off), b = __hsub2(*reinterpret_cast<const __half2 *>(&h), off);
            lo = *reinterpret_cast<const uint32_t *>(&a), hi = *reinterpret_cast<const uint32_t *>(&b);
        }
    }
    __device__ __forceinline__ float ex2(float x) {
        float y;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
        return y;
    }
    __device__ __forceinline__ uint32_t f16x2(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }

    template <typename T> __device__ __forceinline__ uint32_t pair16(float a, float b);
    template <> __device__ __forceinline__ uint32_t pair16<__half>(float a, float b) { return f16x2(a, b); }
    template <> __device__ __forceinline__ uint32_t pair16<__nv_bfloat16>(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }

    // A position on the line: tile `tile` of the `n` tiles of the unit (b, hk).
    struct At {
        int b, hk, tile, n;
    };

    // kUnit: one CTA per unit, its warps take the unit's tiles in turn and meet in shared memory; no line, no workspace, no second kernel.
    template <typename T, int D, int NT, bool kE4m3, bool kUnit>
    __global__ void __launch_bounds__(Stream<D, NT>::W * 32, 1)
        attn_decode_q8_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ StreamParams p) {
        using L          = Stream<D, NT>;
        constexpr int W = L::W, S = L::S, CH = L::CH, MT = L::MT;
        extern __shared__ uint8_t smem_raw[];
        const uint32_t raw  = ptx::smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
        uint8_t       *gb   = smem_raw + (base - raw);
        volatile int  *ctl  = (volatile int *) (gb + L::oCtl);
        int           *tab  = (int *) (gb + L::oTab);
        const int      warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
        const int      Hkv = (int) p.q.Hkv;

        if (threadIdx.x < W * S) {
            ptx::mbar_init(base + L::oBar + 8u * threadIdx.x, 2); // the copies' arrival and the scales'
            ptx::fence_mbar_init();
        }
        if (threadIdx.x == 0) {
            ctl[0] = 0;
            ptx::prefetch_tmap(&tmK);
            ptx::prefetch_tmap(&tmV);
        }
        vkc_grid_dep_wait();
        vkc_grid_dep_launch();
        int  P0 = 0, P1 = 0, quota = 1, run = 0; // this warp's run [P0, P1) of the line, tiles of a run, number of the run
        At   at;                                 // its first tile
        bool ok = true;
        if constexpr (kUnit) {
            at.b = blockIdx.x / Hkv, at.hk = blockIdx.x - at.b * Hkv, at.tile = warp;
            at.n = (int) ((q8_len(p.q, at.b) + kTile - 1) / kTile);
            P1   = at.n > warp ? (at.n - warp + W - 1) / W : 0;
            if (at.n == 0) { // no key: 0 / 0
                for (int i = threadIdx.x; i < p.G * D; i += W * 32) St<T>::st((T *) p.q.O + ((int64_t) at.b * p.q.Hq + at.hk * p.G) * D + i, q8::nan_value());
                return;
            }
            __syncthreads(); // the barriers are set up
        } else {
            // line positions: sequence b begins at tab[b] and has Hkv * ceil(len / 32) tiles
            {
                __shared__ int wsum[W];
                int            sum = 0;
                for (int b0 = 0; b0 < p.B; b0 += W * 32) {
                    const int b = b0 + threadIdx.x;
                    int       n = b < p.B ? (int) ((q8_len(p.q, b) + kTile - 1) / kTile) * Hkv : 0, incl = n;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const int up = __shfl_up_sync(0xffffffffu, incl, o);
                        if (lane >= o) incl += up;
                    }
                    if (lane == 31) wsum[warp] = incl;
                    __syncthreads();
                    int before = sum, all = sum;
#pragma unroll
                    for (int w = 0; w < W; ++w) {
                        if (w < warp) before += wsum[w];
                        all += wsum[w];
                    }
                    if (b < p.B) tab[b] = before + incl - n;
                    sum = all;
                    __syncthreads();
                }
                if (threadIdx.x == 0) tab[p.B] = sum;
            }
            __syncthreads();
            // sequences without a key: 0 / 0
            for (int b = blockIdx.x; b < p.B; b += gridDim.x)
                if (tab[b] == tab[b + 1])
                    for (int i = threadIdx.x; i < (int) p.q.Hq * D; i += W * 32) St<T>::st((T *) p.q.O + (int64_t) b * p.q.Hq * D + i, q8::nan_value());
            // This warp's run [P0, P1) of the line. Neighbouring runs go to different SMs, so that a short line still uses all of them.
            const int total = tab[p.B], runs = (int) gridDim.x * W;
            run   = warp * (int) gridDim.x + (int) blockIdx.x;
            quota = (total + runs - 1) / runs;
            if (quota < kMinTiles) quota = kMinTiles;
            if (blockIdx.x == 0)
                for (int i = threadIdx.x; i <= p.B + 1; i += W * 32) p.line[i] = i <= p.B ? tab[i] : quota;
            const int64_t c0 = (int64_t) run * quota;
            P0 = c0 < total ? (int) c0 : total, P1 = c0 + quota < total ? (int) (c0 + quota) : total;
            if (P0 < P1) {
                int lo = 0, hi = p.B;
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (tab[mid] <= P0) lo = mid;
                    else hi = mid;
                }
                at.b = lo, at.n = (tab[lo + 1] - tab[lo]) / Hkv;
                at.hk = (P0 - tab[lo]) / at.n, at.tile = P0 - tab[lo] - at.hk * at.n;
            }
        }
        if (kUnit || P0 < P1) {
            auto next_unit = [&](At &x) { // to the beginning of the next unit (there is one)
                x.tile = 0;
                if (++x.hk == Hkv) {
                    x.hk = 0;
                    do ++x.b;
                    while (tab[x.b + 1] == tab[x.b]);
                    x.n = (tab[x.b + 1] - tab[x.b]) / Hkv;
                }
            };
            const int      rows_per_tile = kTile * D / 128, rows_per_unit = (int) (p.q.Lmax * D / 128);
            const int      nb = (int) (p.q.Lmax >> p.block_log2);
            const uint32_t ring = base + L::oRing + (uint32_t) warp * S * 2 * L::TILE, bars = base + L::oBar + 8u * (uint32_t) (warp * S);
            float         *sc   = (float *) (gb + L::oSc) + warp * S * 2;
            const uint32_t sc_a = base + L::oSc + (uint32_t) warp * S * 8;

            // Where in a swizzled tile this lane's chunks of the keys g, g + 8, ... (K) and 2t, 2t + 8, ... and 2t + 1, ... (V) begin. Eight
            // keys further the swizzle is the same again, except that for D = 64 (eight keys are four rows of 128 bytes) bit 6 flips.
            auto     swz = [](uint32_t byte) { return byte ^ (((byte >> 7) & 7u) << 4); };
            uint32_t k_at[CH], v_at[2];
#pragma unroll
            for (int c = 0; c < CH; ++c) k_at[c] = swz((uint32_t) g * D + (D == 256 ? (c >> 1) * 8 + (t & 1) + (t >> 1) * 4 + 2 * (c & 1) : t * CH + c) * 16u);
            v_at[0] = swz((uint32_t) (2 * t) * D + g * (D / 8)), v_at[1] = swz((uint32_t) (2 * t + 1) * D + g * (D / 8));

            // ---- producer (lane 0): the tile at `pa` into stage `ps`
            At       pa = at;
            int      left = P1 - P0; // tiles not yet fetched
            int      row0 = (pa.b * Hkv + pa.hk) * rows_per_unit; // the unit's first row of 128 bytes
            uint32_t p_bar = bars, p_dst = ring, p_sc = sc_a;       // of the stage
            auto     fetch = [&]() {
                if (left == 0) return;
                const int row = row0 + pa.tile * rows_per_tile;
                ptx::mbar_expect_tx(p_bar, 2 * L::TILE);
                ptx::tma_load_2d(p_dst, &tmK, 0, row, p_bar);
                ptx::tma_load_2d(p_dst + L::TILE, &tmV, 0, row, p_bar);
                const int64_t si = (int64_t) (pa.b * Hkv + pa.hk) * nb + ((pa.tile * kTile) >> p.block_log2);
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(p_sc), "l"(p.q.ks + si) : "memory");
                asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(p_sc + 4u), "l"(p.q.vs + si) : "memory");
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(p_bar) : "memory");
                p_bar += 8u, p_dst += 2 * L::TILE, p_sc += 8u;
                if (p_bar == bars + 8u * S) p_bar = bars, p_dst = ring, p_sc = sc_a;
                --left;
                if constexpr (kUnit) {
                    pa.tile += W;
                } else if (left > 0 && ++pa.tile == pa.n) {
                    next_unit(pa);
                    row0 = (pa.b * Hkv + pa.hk) * rows_per_unit;
                }
            };
            if (lane == 0)
                for (int i = 0; i < S; ++i) fetch();
            __syncwarp();

            int      stage = 0;
            uint32_t phase = 0;
            for (int todo = kUnit ? 1 : P1 - P0; todo > 0 && ok;) { // one item: the part of a unit in this run
                const int len = (int) q8_len(p.q, at.b), hq0 = at.hk * p.G, first = at.tile;
                const int end = kUnit || at.n - first < todo ? at.n : first + todo; // its tiles: [first, end)
                float     o[NT][MT][4], m[NT], l[NT], fac[NT];
                uint32_t  qa[NT][D / 16][2];
                // Q of this kv head's group: row g (and g + 8) of the A fragments, dims in the order the key chunks are read in
#pragma unroll
                for (int h = 0; h < NT; ++h) {
                    m[h] = -INFINITY, l[h] = 0.f, fac[h] = p.q.scale_log2;
                    const bool have = h * 8 + g < p.G;
                    const T   *qr   = (const T *) p.q.Q + ((int64_t) at.b * p.q.Hq + hq0 + (have ? h * 8 + g : 0)) * D;
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
                        const int chunk = D == 256 ? (c >> 1) * 8 + (t & 1) + (t >> 1) * 4 + 2 * (c & 1) : t * CH + c;
                        uint4     v[2]; // 16 dims
                        // (plain loads, not the read-only path: the kernel before may still have been writing Q when this one started)
                        v[0] = have ? *reinterpret_cast<const uint4 *>(qr + chunk * 16) : make_uint4(0, 0, 0, 0);
                        v[1] = have ? *(reinterpret_cast<const uint4 *>(qr + chunk * 16) + 1) : make_uint4(0, 0, 0, 0);
                        const uint32_t *w = reinterpret_cast<const uint32_t *>(v);
#pragma unroll
                        for (int k = 0; k < 4; ++k) qa[h][c * 4 + k][0] = w[2 * k], qa[h][c * 4 + k][1] = w[2 * k + 1];
                    }
                    if (!std::is_same<T, __half>::value) {
                        // bf16: times the power of two that brings the row's largest value to [2^14, 2^15), exact in f16 for everything down
                        // to 2^-29 of it; the score takes the inverse. A row of zeros, or with infinities, stays as it is.
                        uint32_t top = 0;
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                const uint32_t x = qa[h][k][e], a = (x << 16) & 0x7fffffffu, c = x & 0x7fff0000u;
                                top              = a > top ? a : top;
                                top              = c > top ? c : top;
                            }
                        uint32_t other = __shfl_xor_sync(0xffffffffu, top, 1);
                        top            = other > top ? other : top;
                        other          = __shfl_xor_sync(0xffffffffu, top, 2);
                        top            = other > top ? other : top;
                        const int e  = (int) (top >> 23) - 127;                                   // top in [2^e, 2^(e+1))
                        const int up = top == 0 || top >= 0x7f800000u ? 0 : (14 - e > 126 ? 126 : 14 - e);
                        const float mul = __uint_as_float((uint32_t) (127 + up) << 23);
                        fac[h] *= __uint_as_float((uint32_t) (127 - up) << 23);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)
#pragma unroll
                            for (int i = 0; i < 2; ++i) qa[h][k][i] = f16x2(__uint_as_float(qa[h][k][i] << 16) * mul, __uint_as_float(qa[h][k][i] & 0xffff0000u) * mul);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) o[h][i][0] = o[h][i][1] = o[h][i][2] = o[h][i][3] = 0.f;
                }
                for (int tile = first; tile < end; tile += kUnit ? W : 1) {
                    ok = ptx::mbar_wait(bars + 8u * stage, phase, ctl, p.dev_err);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t sK = ring + (uint32_t) stage * 2 * L::TILE, sV = sK + L::TILE;
                    const float    ks = sc[2 * stage], vs = sc[2 * stage + 1];
                    const int      nv = len - tile * kTile; // valid keys of the tile
                    // scores: four groups of eight keys
                    float s[4][4];
#pragma unroll
                    for (int c = 0; c < CH; ++c) {
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const uint4    kv   = ptx::ld_shared_v4(sK + n * 8 * D + (D == 64 && (n & 1) ? k_at[c] ^ 64u : k_at[c]));
                            const uint32_t w[4] = {kv.x, kv.y, kv.z, kv.w};
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                uint32_t b0, b1;
                                codes_to_f16<kE4m3>(w[k], b0, b1);
                                const uint32_t *q0 = qa[0][c * 4 + k], *q1 = qa[NT - 1][c * 4 + k];
                                if (c == 0 && k == 0) mma16816_first(s[n], q0[0], NT == 1 ? 0u : q1[0], q0[1], NT == 1 ? 0u : q1[1], b0, b1);
                                else mma16816(s[n], q0[0], NT == 1 ? 0u : q1[0], q0[1], NT == 1 ? 0u : q1[1], b0, b1);
                            }
                        }
                    }
                    uint32_t pb[NT][4]; // P^T as B fragments: keys n * 8 + 2t, + 1 of head g (+ 8)
#pragma unroll
                    for (int h = 0; h < NT; ++h) {
                        const float f = fac[h] * ks;
                        float       x[8], mx = -INFINITY;
#pragma unroll
                        for (int n = 0; n < 4; ++n) x[2 * n] = s[n][h * 2] * f, x[2 * n + 1] = s[n][h * 2 + 1] * f;
                        if (nv < kTile) {
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                if ((i >> 1) * 8 + 2 * t + (i & 1) >= nv) x[i] = -INFINITY;
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i]);
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                        // the maximum is raised only when it grows by more than 2^8: P stays below 2^15 in f16
                        const bool raise = mx > m[h] + 8.f || (m[h] == -INFINITY && mx > m[h]);
                        if (__any_sync(0xffffffffu, raise)) {
                            const float a = raise ? ex2(m[h] - mx) : 1.f; // (0 for the first tile)
                            if (raise) m[h] = mx;
                            l[h] *= a;
                            const float a0 = __shfl_sync(0xffffffffu, a, t * 8), a1 = __shfl_sync(0xffffffffu, a, t * 8 + 4); // heads 2t, 2t + 1
#pragma unroll
                            for (int i = 0; i < MT; ++i) o[h][i][0] *= a0, o[h][i][1] *= a1, o[h][i][2] *= a0, o[h][i][3] *= a1;
                        }
                        const float up = 7.f - m[h];
#pragma unroll
                        for (int n = 0; n < 4; ++n) {
                            const float e0 = ex2(x[n * 2] + up), e1 = ex2(x[n * 2 + 1] + up);
                            l[h] += e0 + e1;
                            pb[h][n] = f16x2(e0, e1);
                        }
                    }
                    // O^T += V^T . P^T, 16 keys a step; word w of a thread's bytes holds the dims of two row tiles
                    constexpr int WPT = D / 32; // 4-byte words of a key per thread
#pragma unroll
                    for (int q4 = 0; q4 < (WPT + 3) / 4; ++q4) {
                        constexpr int NW = WPT < 4 ? WPT : 4;
                        uint32_t      x[2][4][NW]; // [step][key][word]
#pragma unroll
                        for (int st = 0; st < 2; ++st)
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t a = sV + (st * 2 + (k >> 1)) * 8 * D + ((D == 64 && (k >> 1) ? v_at[k & 1] ^ 64u : v_at[k & 1]) ^ (q4 * 16u));
                                if (NW == 4) {
                                    const uint4 v = ptx::ld_shared_v4(a);
                                    x[st][k][0] = v.x, x[st][k][1] = v.y, x[st][k][NW - 2] = v.z, x[st][k][NW - 1] = v.w;
                                } else {
                                    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(x[st][k][0]), "=r"(x[st][k][1]) : "r"(a));
                                }
                            }
                        if (nv < kTile) { // the cache behind the last key may hold any bits
#pragma unroll
                            for (int st = 0; st < 2; ++st)
#pragma unroll
                                for (int k = 0; k < 4; ++k)
                                    if (st * 16 + 2 * t + (k & 1) + (k >> 1) * 8 >= nv)
#pragma unroll
                                        for (int w = 0; w < NW; ++w) x[st][k][w] = 0u;
                        }
#pragma unroll
                        for (int w = 0; w < NW; ++w)
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                float d[NT][4];
#pragma unroll
                                for (int st = 0; st < 2; ++st) {
                                    uint32_t a0, a1, a2, a3;
                                    codes_to_f16<kE4m3>(__byte_perm(x[st][0][w], x[st][1][w], half ? 0x7362 : 0x5140), a0, a1);
                                    codes_to_f16<kE4m3>(__byte_perm(x[st][2][w], x[st][3][w], half ? 0x7362 : 0x5140), a2, a3);
#pragma unroll
                                    for (int h = 0; h < NT; ++h) {
                                        if (st == 0) mma16816_first(d[h], a0, a1, a2, a3, pb[h][0], pb[h][1]);
                                        else mma16816(d[h], a0, a1, a2, a3, pb[h][2], pb[h][3]);
                                    }
                                }
                                const int i = (q4 * 4 + w) * 2 + half;
#pragma unroll
                                for (int h = 0; h < NT; ++h)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) o[h][i][e] = fmaf(vs, d[h][e], o[h][i][e]);
                            }
                    }
                    __syncwarp(); // every lane has read the stage
                    if (lane == 0) fetch();
                    if (++stage == S) stage = 0, phase ^= 1;
                }
                if constexpr (kUnit) {
                    // ---- the warps' (m, l, O) meet in the ring's memory: [warp][head][D], then [warp][head] (m, l)
                    float *image = (float *) (gb + L::oRing), *ml = image + W * NT * 8 * D;
                    __syncthreads(); // every tile has been read
#pragma unroll
                    for (int h = 0; h < NT; ++h) {
                        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                        if (t == 0) ml[((warp * NT + h) * 8 + g) * 2] = m[h], ml[((warp * NT + h) * 8 + g) * 2 + 1] = l[h];
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float4 *to = reinterpret_cast<float4 *>(image + ((warp * NT + h) * 8 + 2 * t + e) * D + g * (D / 8));
#pragma unroll
                            for (int i = 0; i < MT / 2; ++i) to[i] = make_float4(o[h][2 * i][e], o[h][2 * i][2 + e], o[h][2 * i + 1][e], o[h][2 * i + 1][2 + e]);
                        }
                    }
                    __syncthreads();
                    for (int i = threadIdx.x; i < p.G * (D / 4); i += W * 32) {
                        const int hd = i * 4 / D, d = i * 4 - hd * D;
                        float     top = -INFINITY, ls = 0.f;
#pragma unroll
                        for (int w = 0; w < W; ++w) top = fmaxf(top, ml[(w * NT * 8 + hd) * 2]);
                        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                        for (int w = 0; w < W; ++w) {
                            const float  mw = ml[(w * NT * 8 + hd) * 2], lw = ml[(w * NT * 8 + hd) * 2 + 1], a = mw == -INFINITY && lw == 0.f ? 0.f : ex2(mw - top);
                            const float4 v  = *reinterpret_cast<const float4 *>(image + (w * NT * 8 + hd) * D + d);
                            ls              = fmaf(lw, a, ls);
                            acc.x = fmaf(v.x, a, acc.x), acc.y = fmaf(v.y, a, acc.y), acc.z = fmaf(v.z, a, acc.z), acc.w = fmaf(v.w, a, acc.w);
                        }
                        const float inv = 1.0f / ls;
                        *reinterpret_cast<uint2 *>((T *) p.q.O + ((int64_t) at.b * p.q.Hq + hq0 + hd) * D + d) =
                            make_uint2(pair16<T>(acc.x * inv, acc.y * inv), pair16<T>(acc.z * inv, acc.w * inv));
                    }
                    break;
                }
                if (!ok) break;
                // ---- the item's rows: a thread holds D / 8 consecutive dims, from g * D / 8 on, of the heads 2t and 2t + 1
                const bool whole = first == 0 && end == at.n;
                const int  slot  = first == 0 ? 1 : 0; // (of a cut unit)
#pragma unroll
                for (int h = 0; h < NT; ++h) {
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
                    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
                    const int64_t prow = ((int64_t) run * 2 + slot) * p.G + h * 8;
                    if (!whole && t == 0 && h * 8 + g < p.G) p.part_ml[(prow + g) * 2] = m[h], p.part_ml[(prow + g) * 2 + 1] = l[h];
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const float inv = 1.0f / __shfl_sync(0xffffffffu, l[h], t * 8 + e * 4);
                        const int   hd  = h * 8 + 2 * t + e;
                        if (hd >= p.G) continue;
                        if (whole) {
                            uint4 *to = reinterpret_cast<uint4 *>((T *) p.q.O + ((int64_t) at.b * p.q.Hq + hq0 + hd) * D + g * (D / 8));
#pragma unroll
                            for (int i = 0; i < MT / 4; ++i) {
                                uint32_t w[4];
#pragma unroll
                                for (int k = 0; k < 4; ++k) w[k] = pair16<T>(o[h][i * 4 + k][e] * inv, o[h][i * 4 + k][2 + e] * inv);
                                to[i] = make_uint4(w[0], w[1], w[2], w[3]);
                            }
                        } else {
                            float4 *to = reinterpret_cast<float4 *>(p.part_o + (prow + 2 * t + e) * D + g * (D / 8));
#pragma unroll
                            for (int i = 0; i < MT / 2; ++i) to[i] = make_float4(o[h][2 * i][e], o[h][2 * i][2 + e], o[h][2 * i + 1][e], o[h][2 * i + 1][2 + e]);
                        }
                    }
                }
                todo -= end - first;
                if (todo > 0) next_unit(at);
            }
        }
        if (ctl[0])
            for (int i = 0; i < 50; ++i) __nanosleep(20000); // aborted: let copies in flight land
    }

    // Joins one head's partials of unit (sequence blockIdx.z, kv head blockIdx.y) if it was cut: slot 1 of the run it begins in, slot 0
    // of the runs behind it. A thread takes four dims over every `groups`-th partial, eight of them on their way at a time; the
    // groups meet in shared memory, in order.
    constexpr int kJoinGroups = 16;
    template <typename T, int D> __global__ void __launch_bounds__(kJoinGroups * D / 4) attn_decode_q8_join_kernel(const StreamParams p) {
        constexpr int U = 8, LANES = D / 4;
        __shared__ float4 so[kJoinGroups][LANES];
        __shared__ float2 sml[kJoinGroups];
        const int b = blockIdx.z, hk = blockIdx.y, hd = blockIdx.x, grp = threadIdx.x / LANES, ln = threadIdx.x % LANES, groups = blockDim.x / LANES;
        vkc_grid_dep_wait();
        vkc_grid_dep_launch();
        const int t0 = p.line[b], t1 = p.line[b + 1], quota = p.line[p.B + 1];
        const int n = (t1 - t0) / (int) p.q.Hkv, off = t0 + hk * n;
        if (n <= 0 || off < 0 || quota < 1) return;
        const int r0 = off / quota, parts = (off + n - 1) / quota - r0 + 1;
        if (parts < 2 || r0 + parts > p.runs) return; // (beyond the runs only if another call writes the same workspace: stay inside it)
        auto   row = [&](int k) { return ((int64_t) (r0 + k) * 2 + (k ? 0 : 1)) * p.G + hd; };
        float  top = -INFINITY, ls = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        auto   merge = [&](const float2 (&ml)[U], const float4 (&v)[U]) {
            float now = top;
#pragma unroll
            for (int u = 0; u < U; ++u) now = fmaxf(now, ml[u].x);
            // (a part whose scores were all NaN has the maximum -inf and the sum NaN, which must stay)
            const float keep = top == -INFINITY && ls == 0.f ? 0.f : ex2(top - now);
            ls *= keep, acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
            top = now;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float a = ml[u].x == -INFINITY && ml[u].y == 0.f ? 0.f : ex2(ml[u].x - now);
                ls            = fmaf(ml[u].y, a, ls);
                acc.x = fmaf(v[u].x, a, acc.x), acc.y = fmaf(v[u].y, a, acc.y), acc.z = fmaf(v[u].z, a, acc.z), acc.w = fmaf(v[u].w, a, acc.w);
            }
        };
        float2 ml[U];
        float4 v[U];
        for (int k0 = grp; k0 < parts; k0 += U * groups) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int  k    = k0 + u * groups;
                const bool have = k < parts;
                ml[u]           = have ? *reinterpret_cast<const float2 *>(p.part_ml + row(k) * 2) : make_float2(-INFINITY, 0.f);
                v[u]            = have ? *reinterpret_cast<const float4 *>(p.part_o + row(k) * D + ln * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            merge(ml, v);
        }
        if (groups > 1) {
            so[grp][ln] = acc;
            if (ln == 0) sml[grp] = make_float2(top, ls);
            __syncthreads();
            if (grp != 0) return;
            top = -INFINITY, ls = 0.f, acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k0 = 0; k0 < groups; k0 += U) {
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const bool have = k0 + u < groups;
                    ml[u]           = have ? sml[k0 + u] : make_float2(-INFINITY, 0.f);
                    v[u]            = have ? so[k0 + u][ln] : make_float4(0.f, 0.f, 0.f, 0.f);
                }
                merge(ml, v);
            }
        }
        const float inv = 1.0f / ls;
        T          *to  = (T *) p.q.O + ((int64_t) b * p.q.Hq + (int64_t) hk * p.G + hd) * D + ln * 4;
        *reinterpret_cast<uint2 *>(to) = make_uint2(pair16<T>(acc.x * inv, acc.y * inv), pair16<T>(acc.z * inv, acc.w * inv));
    }

    // Runs of a launch that can have tiles, and bytes of the workspace: partials of two cut units for each of them, and the line.
    int64_t stream_runs(int64_t B, int64_t Hkv, int64_t Lmax, int64_t D) {
        const int64_t most = kMaxCtas * (D == 256 ? 4 : 8), b = B < kSliceB ? B : kSliceB;
        const int64_t need = (b * Hkv * ((Lmax + kTile - 1) / kTile) + kMinTiles - 1) / kMinTiles;
        return need < most ? need : most;
    }
    size_t stream_ws(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lmax, int64_t D) {
        return (size_t) stream_runs(B, Hkv, Lmax, D) * 2 * (size_t) (Hq / Hkv) * (size_t) (D + 2) * 4 + (kSliceB + 4) * 4;
    }

    template <typename T, int D, int NT, bool kE4m3>
    int launch_stream(vkc_ctx *ctx, const StreamParams &p, int grid, const CUtensorMap &tk, const CUtensorMap &tv, cudaStream_t st) {
        constexpr int smem = (int) Stream<D, NT>::total;
        if (p.unit) {
            auto kern = attn_decode_q8_kernel<T, D, NT, kE4m3, true>;
            if (int rc = vkc_configure_smem(ctx, kern, smem)) return rc;
            vkc_launch(ctx, kern, dim3((unsigned) (p.B * p.q.Hkv)), dim3(Stream<D, NT>::W * 32), smem, st, tk, tv, p);
            return vkc_post_launch(ctx, "attn_decode_q8");
        }
        auto kern = attn_decode_q8_kernel<T, D, NT, kE4m3, false>;
        if (int rc = vkc_configure_smem(ctx, kern, smem)) return rc;
        vkc_launch(ctx, kern, dim3((unsigned) grid), dim3(Stream<D, NT>::W * 32), smem, st, tk, tv, p);
        if (int rc = vkc_post_launch(ctx, "attn_decode_q8")) return rc;
        // groups of the join: as many as give each of them eight partials of a unit, were all sequences of full length
        const int64_t parts  = (int64_t) grid * Stream<D, NT>::W / ((int64_t) p.B * p.q.Hkv);
        int           groups = 1;
        while (groups < kJoinGroups && parts > 8 * groups) groups *= 2;
        vkc_launch(ctx, attn_decode_q8_join_kernel<T, D>, dim3((unsigned) p.G, (unsigned) p.q.Hkv, (unsigned) p.B), dim3((unsigned) (groups * D / 4)), 0, st, p);
        return vkc_post_launch(ctx, "attn_decode_q8_join");
    }
    template <typename T, int D> int pick_stream_form(vkc_ctx *ctx, const StreamParams &p, bool e4m3, int grid, const CUtensorMap &tk, const CUtensorMap &tv, cudaStream_t st) {
        if (p.G <= 8) return e4m3 ? launch_stream<T, D, 1, true>(ctx, p, grid, tk, tv, st) : launch_stream<T, D, 1, false>(ctx, p, grid, tk, tv, st);
        return e4m3 ? launch_stream<T, D, 2, true>(ctx, p, grid, tk, tv, st) : launch_stream<T, D, 2, false>(ctx, p, grid, tk, tv, st);
    }

    // Whether one CTA per unit beats equal runs over all warps, by the cache's length (the sequences' own are on the device): up to four
    // tiles per warp in one round of CTAs, two in two rounds. It saves the line, the partials and the second kernel, but its rounds do
    // not overlap and it does not even out lengths. Measured in a graph, us, unit against runs, D = 128 where not said: 12 units of 512
    // keys at D = 64 4.3 / 6.7, 32 of 1024 7.5 / 7.8, 128 of 1024 7.9 / 12.2, 64 of 512 at D = 256 9.3 / 11.5 (4 of them 9.1 / 8.1, but
    // the call costs the host 1.6 us less), 256 of 512 9.0 / 11.0; beyond: 32 of 1536 9.7 / 8.5, 32 of 2048 11.8 / 8.9, 160 of 1024
    // 16.6 / 15.8, 400 of 512 17.6 / 17.5, 960 of 256 at D = 64 20 / 15.4.
    bool one_cta_per_unit(int64_t B, int64_t Hkv, int64_t Lmax, int64_t D, int sms) {
        const int64_t W = D == 256 ? 4 : 8, rounds = (B * Hkv + sms - 1) / sms;
        return B <= kSliceB && rounds <= 2 && rounds * (Lmax / kTile) <= 4 * W;
    }

    // The tensor-core forms for the whole call, kSliceB sequences per launch.
    int run_stream(vkc_ctx *ctx, const DecQ8Params &q, int64_t B, int64_t D, bool e4m3, int dtype, bool unit, void *ws, cudaStream_t st) {
        const int64_t G = q.Hq / q.Hkv;
        for (int64_t b0 = 0; b0 < B; b0 += kSliceB) {
            StreamParams p;
            p.q = q, p.B = (int) (B - b0 < kSliceB ? B - b0 : kSliceB), p.G = (int) G, p.block_log2 = q.block == 32 ? 5 : q.block == 64 ? 6 : 7;
            const int64_t per = q.Hkv * q.Lmax, cache0 = b0 * per * D, scale0 = b0 * (per / q.block);
            p.q.Q = (const char *) q.Q + b0 * q.Hq * D * 2, p.q.O = (char *) q.O + b0 * q.Hq * D * 2;
            p.q.Kc += cache0, p.q.Vc += cache0, p.q.ks += scale0, p.q.vs += scale0;
            if (q.kv_len) p.q.kv_len += b0;
            p.dev_err = ctx->dev_err;
            // one CTA per SM, or one for each run where there are fewer (a CTA's runs are spread over the line, so that the others
            // of its warps are then idle)
            const int64_t runs = stream_runs(B, q.Hkv, q.Lmax, D), here = stream_runs(p.B, q.Hkv, q.Lmax, D);
            int64_t       grid = ctx->sm_count < kMaxCtas ? ctx->sm_count : kMaxCtas;
            if (grid > here) grid = here;
            p.runs    = (int) runs;
            p.unit    = unit;
            p.part_o  = (float *) ws;
            p.part_ml = p.part_o + runs * 2 * G * D;
            p.line    = (int *) (p.part_ml + runs * 2 * G * 2);
            // both caches as rows of 128 bytes, whatever D is
            CUtensorMap    tk, tv;
            const uint64_t dims[2] = {64, (uint64_t) (p.B * per * D / 128)}, stride[1] = {128};
            const uint32_t box[2]  = {64, (uint32_t) (kTile * D / 128)};
            if (int rc = vkc_make_tmap(ctx, &tk, VKC_F16, p.q.Kc, 2, dims, stride, box)) return rc;
            if (int rc = vkc_make_tmap(ctx, &tv, VKC_F16, p.q.Vc, 2, dims, stride, box)) return rc;
            int rc;
            if (dtype == VKC_F16)
                rc = D == 64 ? pick_stream_form<__half, 64>(ctx, p, e4m3, (int) grid, tk, tv, st) : D == 128 ? pick_stream_form<__half, 128>(ctx, p, e4m3, (int) grid, tk, tv, st)
                                                                                                       : pick_stream_form<__half, 256>(ctx, p, e4m3, (int) grid, tk, tv, st);
            else
                rc = D == 64 ? pick_stream_form<__nv_bfloat16, 64>(ctx, p, e4m3, (int) grid, tk, tv, st)
                             : D == 128 ? pick_stream_form<__nv_bfloat16, 128>(ctx, p, e4m3, (int) grid, tk, tv, st)
                                        : pick_stream_form<__nv_bfloat16, 256>(ctx, p, e4m3, (int) grid, tk, tv, st);
            if (rc) return rc;
        }
        return VKC_OK;
    }

    template <typename T, int D> void launch_simt(vkc_ctx *ctx, bool e4m3, dim3 grid, cudaStream_t st, const DecQ8Params &p) {
        if (e4m3) vkc_launch(ctx, attn_decode_q8_simt_kernel<T, D, true>, grid, dim3(kSimtWarps * 32), 0, st, p);
        else vkc_launch(ctx, attn_decode_q8_simt_kernel<T, D, false>, grid, dim3(kSimtWarps * 32), 0, st, p);
    }

} // namespace

extern "C" size_t vkc_attn_decode_q8_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t Lmax, int64_t D) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || Lmax <= 0 || D <= 0) return 0;
    return stream_ws(B, Hq, Hkv, Lmax, D);
}

extern "C" int vkc_attn_decode_q8(vkc_ctx *ctx, const vkc_attn_decode_q8_args *args, vkc_stream stream) {
    if (!ctx) return VKC_ERR_INVALID;
    VKC_REQUIRE(ctx, args, "attn_decode_q8: null arguments");
    const auto [Q, Kc, Vc, k_scale, v_scale, O, B, Hq, Hkv, Lmax, D, block, kv_len, given, workspace_bytes, scale, dtype, cache_dtype] = *args;
    void *workspace = given;
    VKC_REQUIRE(ctx, B >= 0 && Hq >= 1 && Hkv >= 1 && Lmax >= 1 && D >= 1, "attn_decode_q8: bad extents");
    VKC_REQUIRE(ctx, Hq % Hkv == 0, "attn_decode_q8: Hq=%lld is not a multiple of Hkv=%lld", (long long) Hq, (long long) Hkv);
    if (dtype != VKC_F16 && dtype != VKC_BF16) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "attn_decode_q8: Q and O must be f16 or bf16");
    if (int rc = vkc_q8_check(ctx, "attn_decode_q8", B, Hkv, Lmax, D, block, cache_dtype)) return rc;
    VKC_REQUIRE(ctx, Hq <= 65535 * 16, "attn_decode_q8: extents too large");
    if (B == 0) return VKC_OK;
    VKC_REQUIRE(ctx, Q && Kc && Vc && k_scale && v_scale && O, "attn_decode_q8: null tensor");
    VKC_REQUIRE(ctx, !(((uintptr_t) Q | (uintptr_t) O | (uintptr_t) Kc | (uintptr_t) Vc) & 15), "attn_decode_q8: Q, O and the cache must be 16-byte aligned");
    VKC_REQUIRE(ctx, !(((uintptr_t) k_scale | (uintptr_t) v_scale | (uintptr_t) kv_len) & 3), "attn_decode_q8: scales or lengths are not aligned to their type");
    const size_t need = vkc_attn_decode_q8_workspace_bytes(B, Hq, Hkv, Lmax, D);
    VKC_REQUIRE(ctx, !workspace || (workspace_bytes >= need && !((uintptr_t) workspace & 15)),
                "attn_decode_q8: workspace of %zu bytes is smaller than the %zu required, or not 16-byte aligned", workspace_bytes, need);
    VkcDeviceGuard guard(ctx);
    cudaStream_t   st = vkc_pick_stream(ctx, stream);
    DecQ8Params    p;
    p.Q = Q, p.Kc = (const uint8_t *) Kc, p.Vc = (const uint8_t *) Vc, p.ks = k_scale, p.vs = v_scale, p.O = O;
    p.Hq = Hq, p.Hkv = Hkv, p.Lmax = Lmax, p.block = (int) block, p.kv_len = kv_len;
    p.scale_log2 = scale * 1.4426950408889634f;
    const dim3 grid((unsigned) Hq, (unsigned) B);
    const bool e4m3 = cache_dtype == VKC_E4M3;
    // The streaming form holds a group of up to 16 query heads and counts line positions and 128-byte rows in 32 bits.
    const bool fits = Hq / Hkv <= 16 && (B < kSliceB ? B : kSliceB) * Hkv * (Lmax / kTile) < INT32_MAX / 2 && (B < kSliceB ? B : kSliceB) * Hkv * Lmax * (D / 64) < INT32_MAX;
    if (fits && ctx->impl != VKC_IMPL_SIMT) {
        const bool unit = one_cta_per_unit(B, Hkv, Lmax, D, ctx->sm_count);
        if (!workspace && !unit) {
            if (int rc = vkc_ensure_scratch(ctx, need, st)) return rc;
            workspace = ctx->scratch;
        }
        return run_stream(ctx, p, B, D, e4m3, dtype, unit, workspace, st);
    }
    if (ctx->impl == VKC_IMPL_TCGEN05) return vkc_fail(ctx, VKC_ERR_UNSUPPORTED, "attn_decode_q8: more than 16 query heads per kv head, or too large a cache, for the tensor-core form");
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
