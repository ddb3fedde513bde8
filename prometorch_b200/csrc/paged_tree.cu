// Rows of drafted tokens against a paged cache on mma.sync, and the merge of items that were cut; see paged_tree.cuh.
//
// One CTA per SM.  Warp 8 brings pages: keys and values of a (page, kv head), each one TMA box of 128-byte rows with the 128-byte swizzle, through a ring deep enough
// to cover the memory's latency on its own.  Eight warps compute: RG groups of 16 rows times KG = 8 / RG groups of 16-token pieces of a page.  Each warp keeps
// an online softmax of its own over its tokens and joins the others when an item ends.
//
// S = Q K^T and O = P V are m16n8k16 products whose operands come from shared memory 16 bytes a lane, without a transposing load.  The order of the contraction is
// free as long as both operands keep it, so lane c of a row's four holds whole 16-byte pieces of a key; and output column n of tile t may
// be any head element, so lane r holds one 16-byte piece of a value row for all tiles.  Which of eight tokens lane r takes (`token_of`) is chosen so
// that the eight lanes of a quarter warp fall on the eight 16-byte columns of the swizzled rows, for keys and for values.
//
// e4m3 pages: values become fp16 exactly, queries are scaled by a power of two into fp16 (they come with eight bits), the exponent of a key's row scales its
// scores, that of a value's row is added to them: p' = 2^(s + e_v) <= 1 weighs the raw e4m3 values, and the sum takes p' 2^-e_v.  P is rounded to the operand's
// type (by at most 2^-11 of a weight in fp16, 2^-8 in bf16, without a bias); scores, maxima, sums and accumulators are fp32.
#include "paged_tree.cuh"

namespace ptb {
namespace tree {
namespace {

constexpr int WARPS = 8, THREADS = (WARPS + 1) * 32;

// Geometry of a page of one head, as 128-byte rows.
template <int D, bool Q8>
struct Geo {
    static constexpr int ROW = D * (Q8 ? 1 : 2);                       // bytes of a token
    static constexpr int BYTES = PAGE * ROW, LINES = BYTES / 128;
    static constexpr int STAGE = 2 * BYTES + (Q8 ? 1024 : 0);          // keys, values, exponents of both
    static constexpr int KSTEPS = D / 16, VTILES = D / 8;
    static constexpr int STAGES = (128 * 1024) / (2 * BYTES) < 12 ? (128 * 1024) / (2 * BYTES) : 12;
    static constexpr int PITCH = D + 8;                                // floats of a row of the joining buffer
};

template <int D, bool Q8, int RG>
struct Sm {
    using G = Geo<D, Q8>;
    static constexpr int KG = WARPS / RG, ROWS = 16 * RG;
    static constexpr int OFF_JOIN = G::STAGES * G::STAGE;
    static constexpr int OFF_ML = OFF_JOIN + KG * ROWS * G::PITCH * 4, OFF_BAR = OFF_ML + KG * ROWS * 8, OFF_PLAN = OFF_BAR + 512;
    static constexpr int TOTAL = OFF_PLAN + 1024;                      // and (B + 1) ints
    static_assert(TOTAL + MAX_B * 4 + 4 <= 227 * 1024, "shared memory of a CTA");
};

// Which of eight neighbouring tokens lane r (0 .. 7) takes; see above.  Keys: lanes 2p and 2p + 1 of one phase differ in the bit that moves a token to the other
// half of a line.  Values: the tokens of lanes 0, 2, 4, 6 (and of 1, 3, 5, 7) fall on four different pairs of columns.
template <int ROW>
__device__ __forceinline__ int token_of(int r) {
    constexpr uint32_t order = ROW == 128 ? 0x37156240u : ROW == 256 ? 0x57463120u : 0x65742130u;
    return (order >> (4 * r)) & 7;
}
// Offset of byte `at` of token t in a swizzled page.
template <int ROW>
__device__ __forceinline__ uint32_t place(int t, int at) {
    const uint32_t x = t * ROW + at;
    return x ^ (((x >> 7) & 7) << 4);
}

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(a));
    return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t a) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
    return v;
}
// Two e4m3 values (the low 16 bits) as fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t two) {
    uint32_t h;
    asm("{\n .reg .b16 lo;\n cvt.u16.u32 lo, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(h) : "r"(two));
    return h;
}
template <bool Q8>
__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    if constexpr (Q8)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <bool Q8>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if constexpr (Q8) { const __half2 h = __floats2half2_rn(x, y); memcpy(&r, &h, 4); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); memcpy(&r, &h, 4); }
    return r;
}
__device__ __forceinline__ void join_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)),
                 "r"(c0), "r"(c1)
                 : "memory");
}

// Head element of contraction step s, lane c (the first of four), and of output tile t, column n.
template <int D, bool Q8>
__device__ __forceinline__ constexpr int k_elem(int s, int c) {
    return Q8 ? (D == 128 ? (s / 4) * 64 + c * 16 + (s % 4) * 4 : c * 16 + s * 4) : (s / 4) * 64 + (c + 4 * ((s / 2) & 1)) * 8 + (s & 1) * 4;
}
template <int D, bool Q8>
__device__ __forceinline__ constexpr int v_elem(int t, int n) {
    return Q8 ? n * (D / 8) + t : (t / 8) * 64 + n * 8 + t % 8;
}

// Where a CTA's run stands.
struct Item { int b, tile, kvh, first, pages, unit0; Req r; };       // first: the page its part begins with; unit0: the item's first unit
__device__ __forceinline__ Item item_at(const Params& P, const int* starts, int u) {
    int lo = 0, hi = P.B;                                // the last request that starts at or before u (empty ones share a start with the next)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= u) lo = mid; else hi = mid;
    }
    Item it;
    it.b = lo;
    it.r = req_of(P, lo);
    it.pages = it.r.pages;
    const int in = u - starts[lo], i = in / it.pages;
    it.first = in - i * it.pages;
    it.tile = i / P.Hk;
    it.kvh = i - it.tile * P.Hk;
    it.unit0 = u - it.first;
    return it;
}

template <int D, bool Q8, int RG>
__global__ void __launch_bounds__(THREADS, 1) paged_tree_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params P) {
    using Ge = Geo<D, Q8>;
    using S = Sm<D, Q8, RG>;
    constexpr int KG = S::KG, ROWS = S::ROWS, ROW = Ge::ROW;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* joined = reinterpret_cast<float*>(smem + S::OFF_JOIN);
    float2* ml = reinterpret_cast<float2*>(smem + S::OFF_ML);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
    uint64_t* empty = full + Ge::STAGES;
    int* bad_page = reinterpret_cast<int*>(empty + Ge::STAGES);        // [STAGES]
    int* part = bad_page + Ge::STAGES;                                 // [9]
    int* starts = reinterpret_cast<int*>(smem + S::OFF_PLAN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // a stage is read by all eight warps, or, with eight groups of tokens and four pieces a page, by four
    constexpr int READERS = KG == 8 ? 4 : 8;
    if (threadIdx.x == 0) {
        for (int s = 0; s < Ge::STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], READERS); }
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    plan<THREADS>(P, starts, part);
    __syncthreads();
    const int all = starts[P.B], per = units_per_cta(all, P.ctas);
    const int u0 = (int)min((long long)all, (long long)blockIdx.x * per), u1 = min(all, u0 + per);
    if (u0 >= u1) return;

    if (warp == WARPS) {
        // ------------------------------------------------------------------------------------ pages
        bool ok = true;
        int u = u0, it_n = 0;
        while (u < u1 && ok) {
            const Item it = item_at(P, starts, u);
            const int n = min(it.pages - it.first, u1 - u);
            for (int p0 = 0; p0 < n && ok; p0 += 32) {   // page ids 32 at a time
                int id = -1;
                if (p0 + lane < n) {
                    id = P.page_table[(size_t)it.b * P.pt_stride + it.first + p0 + lane];
                    if (id < 0 || id >= P.n_pages) {
                        id = -1;
                        if (P.status) atomicExch(P.status, PTB_ERR_BOUNDS);
                    }
                }
                for (int p = 0; p < min(32, n - p0) && ok; ++p, ++it_n) {
                    const int page = __shfl_sync(0xffffffffu, id, p), s = it_n % Ge::STAGES;
                    if (it_n >= Ge::STAGES) ok = mbar_wait(&empty[s], (uint32_t)((it_n / Ge::STAGES - 1) & 1), P.status);
                    if (ok && lane == 0) {
                        bad_page[s] = page < 0;
                        if (page < 0) {
                            mbar_arrive(&full[s]);
                        } else {
                            uint8_t* st = smem + s * Ge::STAGE;
                            const int head = page * P.Hk + it.kvh;
                            mbar_expect_tx(&full[s], 2 * Ge::BYTES + (Q8 ? 2 * PAGE : 0));
                            tma_2d(st, &tmK, 0, head * Ge::LINES, &full[s]);
                            tma_2d(st + Ge::BYTES, &tmV, 0, head * Ge::LINES, &full[s]);
                            if (Q8) {
                                bulk_g2s(st + 2 * Ge::BYTES, P.k_exp + (size_t)head * PAGE, PAGE, &full[s]);
                                bulk_g2s(st + 2 * Ge::BYTES + PAGE, P.v_exp + (size_t)head * PAGE, PAGE, &full[s]);
                            }
                        }
                    }
                    ok = __all_sync(0xffffffffu, ok);
                }
            }
            u += n;
        }
        return;                                          // the warps below wait for every copy it started
    }

    // ---------------------------------------------------------------------------------------- rows
    const int rg = warp % RG, kg = warp / RG, r = lane >> 2, c = lane & 3;
    int it_n = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
        const Item it = item_at(P, starts, u);
        const int n = min(it.pages - it.first, u1 - u), len = it.r.len, total = len + it.r.nodes;
        // this lane's two rows
        uint32_t qa[Ge::KSTEPS][4];
        float fac[2];
        unsigned long long seen[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = it.tile * ROWS + rg * 16 + r + 8 * x, node = row / P.G, g = row - node * P.G;
            const bool on = node < it.r.nodes;
            seen[x] = !on ? 0ull : P.mask ? P.mask[(size_t)it.b * P.T + node] : node == 63 ? ~0ull : (2ull << node) - 1;
            const __nv_bfloat16* q = P.q + (size_t)it.b * P.q_batch + (size_t)(on ? node : 0) * P.q_row + (size_t)(it.kvh * P.G + g) * D;
            uint2 raw[Ge::KSTEPS];
#pragma unroll
            for (int s = 0; s < Ge::KSTEPS; ++s) raw[s] = on ? *reinterpret_cast<const uint2*>(q + k_elem<D, Q8>(s, c)) : make_uint2(0, 0);
            fac[x] = P.scale_log2;
            if constexpr (Q8) {                          // the row's largest magnitude to [1, 2)
                uint32_t a = 0;
#pragma unroll
                for (int s = 0; s < Ge::KSTEPS; ++s)
                    a = max(a, max(max(raw[s].x & 0x7fffu, (raw[s].x >> 16) & 0x7fffu), max(raw[s].y & 0x7fffu, (raw[s].y >> 16) & 0x7fffu)));
                a = max(a, __shfl_xor_sync(0xffffffffu, a, 1));
                a = max(a, __shfl_xor_sync(0xffffffffu, a, 2));
                const int k = min(253, max(1, (int)(a >> 7)));               // biased exponent
                const float down = __uint_as_float((uint32_t)(254 - k) << 23);
                fac[x] *= __uint_as_float((uint32_t)k << 23);
#pragma unroll
                for (int s = 0; s < Ge::KSTEPS; ++s) {
                    const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[s].x)), hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw[s].y));
                    qa[s][x] = pack2<true>(lo.x * down, lo.y * down);
                    qa[s][2 + x] = pack2<true>(hi.x * down, hi.y * down);
                }
            } else {
#pragma unroll
                for (int s = 0; s < Ge::KSTEPS; ++s) { qa[s][x] = raw[s].x; qa[s][2 + x] = raw[s].y; }
            }
        }
        float acc[Ge::VTILES][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < Ge::VTILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

        for (int p = 0; p < n; ++p, ++it_n) {
            const int s = it_n % Ge::STAGES;
            if (KG == 8 && (kg >> 2) != (it_n & 1)) continue;            // every other page
            if (ok) ok = mbar_wait(&full[s], (uint32_t)((it_n / Ge::STAGES) & 1), P.status);
            const int page0 = (it.first + p) * PAGE;
            if (ok && !bad_page[s]) {
                const uint32_t sk = smem_u32(smem + s * Ge::STAGE), sv = sk + Ge::BYTES, se = sv + Ge::BYTES;
                const bool tail = page0 + PAGE > len;    // some of its tokens are drafted, or lie behind the last
#pragma unroll 1
                for (int piece = kg % 4; piece < 4; piece += KG < 4 ? KG : 4) {
                    const int t0 = piece * 16;
                    if (page0 + t0 >= total) break;
                    float sc[2][4];
                    float ev[2][2], un[2][2];            // exponent of a token's values, 2^-exponent
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[j][i] = 0.f;
                        const int kt = t0 + 8 * j + token_of<ROW>(r);
                        if constexpr (Q8) {
#pragma unroll
                            for (int h = 0; h < D / 64; ++h) {
                                const uint4 w = lds128(sk + place<ROW>(kt, h * 64 + c * 16));
                                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                                for (int i = 0; i < 4; ++i) mma<true>(sc[j], qa[h * 4 + i], e4m3x2(ww[i]), e4m3x2(ww[i] >> 16));
                            }
                        } else {
#pragma unroll
                            for (int h = 0; h < D / 32; ++h) {
                                const uint4 w = lds128(sk + place<ROW>(kt, (h >> 1) * 128 + (c + 4 * (h & 1)) * 16));
                                mma<false>(sc[j], qa[2 * h], w.x, w.y);
                                mma<false>(sc[j], qa[2 * h + 1], w.z, w.w);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            const int t = t0 + 8 * j + token_of<ROW>(2 * c + y);
                            float ks = 1.f;
                            ev[j][y] = 0.f;
                            un[j][y] = 1.f;
                            if constexpr (Q8) {
                                // a byte of a slot that nobody wrote may hold any exponent: clamped to what is ever stored
                                const int ke = min(191, max(63, (int)lds8(se + t))), ve = min(191, max(63, (int)lds8(se + PAGE + t)));
                                ks = __uint_as_float((uint32_t)ke << 23);
                                ev[j][y] = (float)(ve - 127);
                                un[j][y] = __uint_as_float((uint32_t)(254 - ve) << 23);
                            }
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                float& v = sc[j][2 * x + y];
                                if constexpr (Q8) v = fmaf(v * ks, fac[x], ev[j][y]);
                                else v *= fac[x];
                                if (tail) {
                                    const int d = page0 + t - len;
                                    if (d >= 0 && (d >= it.r.nodes || !((seen[x] >> d) & 1))) v = -INFINITY;
                                }
                            }
                        }
                    float mx[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        mx[x] = fmaxf(fmaxf(sc[0][2 * x], sc[0][2 * x + 1]), fmaxf(sc[1][2 * x], sc[1][2 * x + 1]));
                        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 1));
                        mx[x] = fmaxf(mx[x], __shfl_xor_sync(0xffffffffu, mx[x], 2));
                    }
                    if (__any_sync(0xffffffffu, mx[0] > m[0] || mx[1] > m[1])) {
                        float f[2];
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            const float mn = fmaxf(m[x], mx[x]);
                            f[x] = mn == -INFINITY ? 1.f : exp2f(m[x] - mn);
                            m[x] = mn;
                            l[x] *= f[x];
                        }
#pragma unroll
                        for (int t = 0; t < Ge::VTILES; ++t) { acc[t][0] *= f[0]; acc[t][1] *= f[0]; acc[t][2] *= f[1]; acc[t][3] *= f[1]; }
                    }
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float mu = m[x] == -INFINITY ? 0.f : m[x];
#pragma unroll
                        for (int j = 0; j < 2; ++j)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                float& v = sc[j][2 * x + y];
                                v = exp2f(v - mu);
                                l[x] = Q8 ? fmaf(v, un[j][y], l[x]) : l[x] + v;
                            }
                    }
                    const uint32_t pa[4] = {pack2<Q8>(sc[0][0], sc[0][1]), pack2<Q8>(sc[0][2], sc[0][3]), pack2<Q8>(sc[1][0], sc[1][1]), pack2<Q8>(sc[1][2], sc[1][3])};
                    // values of this lane's four tokens
                    constexpr int VW = D * (Q8 ? 1 : 2) / 32;            // words of a lane's piece(s) of a value row
                    uint32_t vw[4][VW];
                    bool odd = false;                    // a value that is no number, which a row that does not see its token must not meet
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int t = t0 + 8 * (k >> 1) + token_of<ROW>(2 * c + (k & 1));
                        if constexpr (Q8 && D == 64) {
                            const uint2 w = lds64(sv + place<ROW>(t, r * 8));
                            vw[k][0] = w.x; vw[k][1] = w.y;
                        } else {
#pragma unroll
                            for (int h = 0; h < VW / 4; ++h) {
                                const uint4 w = lds128(sv + place<ROW>(t, h * 128 + r * 16));
                                vw[k][4 * h] = w.x; vw[k][4 * h + 1] = w.y; vw[k][4 * h + 2] = w.z; vw[k][4 * h + 3] = w.w;
                            }
                        }
                        if (tail) {
                            const int d = page0 + t - len;
                            if (d >= it.r.nodes) {
#pragma unroll
                                for (int i = 0; i < VW; ++i) vw[k][i] = 0;
                            } else if (d >= 0) {
#pragma unroll
                                for (int i = 0; i < VW; ++i) {
                                    if constexpr (Q8) odd |= __vcmpeq4(vw[k][i] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0;
                                    else odd |= __vcmpeq2(vw[k][i] & 0x7f807f80u, 0x7f807f80u) != 0;
                                }
                            }
                        }
                    }
                    if (!tail || !__any_sync(0xffffffffu, odd)) {
                        if constexpr (Q8) {
#pragma unroll
                            for (int i = 0; i < VW; ++i) {
                                const uint32_t a0 = __byte_perm(vw[0][i], vw[1][i], 0x5140), a1 = __byte_perm(vw[0][i], vw[1][i], 0x7362);
                                const uint32_t b0 = __byte_perm(vw[2][i], vw[3][i], 0x5140), b1 = __byte_perm(vw[2][i], vw[3][i], 0x7362);
                                mma<true>(acc[4 * i], pa, e4m3x2(a0), e4m3x2(b0));
                                mma<true>(acc[4 * i + 1], pa, e4m3x2(a0 >> 16), e4m3x2(b0 >> 16));
                                mma<true>(acc[4 * i + 2], pa, e4m3x2(a1), e4m3x2(b1));
                                mma<true>(acc[4 * i + 3], pa, e4m3x2(a1 >> 16), e4m3x2(b1 >> 16));
                            }
                        } else {
#pragma unroll
                            for (int i = 0; i < VW; ++i) {
                                mma<false>(acc[2 * i], pa, __byte_perm(vw[0][i], vw[1][i], 0x5410), __byte_perm(vw[2][i], vw[3][i], 0x5410));
                                mma<false>(acc[2 * i + 1], pa, __byte_perm(vw[0][i], vw[1][i], 0x7632), __byte_perm(vw[2][i], vw[3][i], 0x7632));
                            }
                        }
                    } else {                             // token by token, each for the rows that see it
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            // token k: accumulator element (k / 8, y) of lane r * 4 + k % 8 / 2
                            const int t = t0 + (k & 8) + token_of<ROW>(k & 7), from = (lane & ~3) | ((k & 7) >> 1), d = page0 + t - len;
                            const float w0 = __shfl_sync(0xffffffffu, sc[k >> 3][k & 1], from), w1 = __shfl_sync(0xffffffffu, sc[k >> 3][2 + (k & 1)], from);
                            if (d >= it.r.nodes) continue;
                            const bool s0 = d < 0 || ((seen[0] >> d) & 1), s1 = d < 0 || ((seen[1] >> d) & 1);
#pragma unroll 1
                            for (int y = 0; y < 2; ++y)
#pragma unroll
                                for (int tt = 0; tt < Ge::VTILES; ++tt) {
                                    const int e = v_elem<D, Q8>(tt, 2 * c + y);
                                    float v;
                                    if constexpr (Q8) v = __half2float(__ushort_as_half((unsigned short)(e4m3x2(lds8(sv + place<ROW>(t, e))) & 0xffff)));
                                    else v = __uint_as_float(lds16(sv + place<ROW>(t, 2 * e)) << 16);
                                    if (s0) { if (y) acc[tt][1] += w0 * v; else acc[tt][0] += w0 * v; }
                                    if (s1) { if (y) acc[tt][3] += w1 * v; else acc[tt][2] += w1 * v; }
                                }
                        }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
        }
        // ---- the item ends here, or the run does: join the warps' parts
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            const int row = rg * 16 + r + 8 * x;
            if (c == 0) ml[kg * ROWS + row] = make_float2(m[x], l[x]);
            float* dst = joined + (size_t)(kg * ROWS + row) * Ge::PITCH + 2 * c;
#pragma unroll
            for (int t = 0; t < Ge::VTILES; ++t) *reinterpret_cast<float2*>(dst + 8 * t) = make_float2(acc[t][2 * x], acc[t][2 * x + 1]);
        }
        join_sync();
        const bool whole = n == it.pages;
        const int slot = u == u0 ? 0 : 1;
        float* wk = P.work + partial_at(P, blockIdx.x, slot, D);
        for (int e = threadIdx.x; e < ROWS * D / 2; e += WARPS * 32) {       // two elements a thread
            const int row = e / (D / 2), i = (e - row * (D / 2)) * 2;
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < KG; ++k) M = fmaxf(M, ml[k * ROWS + row].x);
            float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
            for (int k = 0; k < KG; ++k) {
                const float2 q = ml[k * ROWS + row];
                const float f = q.x == -INFINITY ? 0.f : exp2f(q.x - M);
                const float2 a = *reinterpret_cast<const float2*>(joined + (size_t)(k * ROWS + row) * Ge::PITCH + i);
                L += q.x == -INFINITY ? 0.f : q.y * f;
                o0 += q.x == -INFINITY ? 0.f : a.x * f;
                o1 += q.x == -INFINITY ? 0.f : a.y * f;
            }
            // place i of a row: column i % 8 of tile i / 8
            if (whole) {
                const int at = it.tile * ROWS + row, node = at / P.G, g = at - node * P.G;
                if (node < P.T) {
                    const bool on = node < it.r.nodes && L != 0.f;
                    __nv_bfloat16* o = P.out + (((size_t)it.b * P.T + node) * P.H + it.kvh * P.G + g) * D;
                    o[v_elem<D, Q8>(i / 8, i % 8)] = __float2bfloat16_rn(on ? o0 / L : 0.f);
                    o[v_elem<D, Q8>(i / 8, i % 8 + 1)] = __float2bfloat16_rn(on ? o1 / L : 0.f);
                }
            } else {
                *reinterpret_cast<float2*>(wk + (size_t)row * D + i) = make_float2(o0, o1);
                if (i == 0) *reinterpret_cast<float2*>(wk + (size_t)ROWS * D + 2 * row) = make_float2(M, L);
            }
        }
        join_sync();                                     // the buffer is free again
        u += n;
    }
}

// Items that several CTAs share: one block per (sixteen rows of an item, 32 columns); and the rows that no unit belongs to, which are zeros.
constexpr int MERGE_THREADS = 256;
template <int D, bool Q8>
__global__ void __launch_bounds__(MERGE_THREADS) paged_tree_merge_kernel(const __grid_constant__ Params P) {
    __shared__ int part[2][MERGE_THREADS / 32];
    __shared__ float fac[16][17];
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, per_item = P.tile_rows / 16 * (D / 32);
    const int i = blockIdx.x / per_item, sub = blockIdx.x - i * per_item, row0 = sub / (D / 32) * 16, col0 = sub % (D / 32) * 32;
    const int tile = i / P.Hk, kvh = i - tile * P.Hk;
    const Req r = req_of(P, b);
    // this request's first unit, and all units
    int before = 0, all = 0;
    for (int x = threadIdx.x; x < P.B; x += MERGE_THREADS) {
        const int u = units_of(P, req_of(P, x));
        all += u;
        if (x < b) before += u;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) { before += __shfl_xor_sync(0xffffffffu, before, o); all += __shfl_xor_sync(0xffffffffu, all, o); }
    if ((threadIdx.x & 31) == 0) { part[0][threadIdx.x >> 5] = before; part[1][threadIdx.x >> 5] = all; }
    __syncthreads();
    before = all = 0;
    for (int w = 0; w < MERGE_THREADS / 32; ++w) { before += part[0][w]; all += part[1][w]; }
    const bool empty = tile >= r.tiles;
    const int per = units_per_cta(all, P.ctas), a = before + i * r.pages, e = a + r.pages;
    const int c0 = empty ? 0 : a / per, c1 = empty ? 0 : (e - 1) / per;
    if (!empty && c0 == c1) return;                      // written already
    const int row = threadIdx.x / 16, col = col0 + (threadIdx.x % 16) * 2, at = tile * P.tile_rows + row0 + row, node = at / P.G, g = at - node * P.G;
    float o0 = 0.f, o1 = 0.f, L = 0.f, M = -INFINITY;
    if (!empty) {
        auto partial = [&](int c) { return P.work + partial_at(P, c, c * per >= a ? 0 : 1, D); };     // slot 0: the run begins in (or with) this item
        for (int k0 = c0; k0 <= c1; k0 += 16) {          // sixteen parts at a time: thread (row, k) fetches one maximum
            const int k = k0 + threadIdx.x % 16;
            __syncthreads();
            float2 ml = make_float2(-INFINITY, 0.f);
            if (k <= c1) ml = *reinterpret_cast<const float2*>(partial(k) + (size_t)P.tile_rows * D + 2 * (row0 + row));
            float mx = ml.x;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            const float mn = fmaxf(M, mx), old = M == -INFINITY ? 0.f : exp2f(M - mn), f = ml.x == -INFINITY ? 0.f : exp2f(ml.x - mn);
            float s = ml.x == -INFINITY ? 0.f : ml.y * f;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            L = L * old + s;
            o0 *= old;
            o1 *= old;
            M = mn;
            fac[row][threadIdx.x % 16] = f;
            __syncwarp();
            for (int x = 0; x < 16 && k0 + x <= c1; ++x) {
                const float w = fac[row][x];
                const float2 v = *reinterpret_cast<const float2*>(partial(k0 + x) + (size_t)(row0 + row) * D + col);
                o0 += v.x * w;
                o1 += v.y * w;
            }
        }
    }
    if (node >= P.T) return;
    const bool on = node < r.nodes && L != 0.f;
    __nv_bfloat16* o = P.out + (((size_t)b * P.T + node) * P.H + kvh * P.G + g) * D;
    o[v_elem<D, Q8>(col / 8, col % 8)] = __float2bfloat16_rn(on ? o0 / L : 0.f);
    o[v_elem<D, Q8>(col / 8, col % 8 + 1)] = __float2bfloat16_rn(on ? o1 / L : 0.f);
}

template <int D, bool Q8, int RG>
int launch(const Params& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
    using S = Sm<D, Q8, RG>;
    static bool attr[64];
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        PTB_CUDA_OK(cudaFuncSetAttribute(paged_tree_kernel<D, Q8, RG>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL + MAX_B * 4 + 4));
        if (dev < 64) attr[dev] = true;
    }
    PTB_CUDA_OK(ptb_launch(paged_tree_kernel<D, Q8, RG>, dim3(p.ctas), dim3(THREADS), (size_t)S::TOTAL + (p.B + 1) * 4, st, ptb_pdl_enabled(), mk, mv, p));
    PTB_CUDA_OK(ptb_launch(paged_tree_merge_kernel<D, Q8>, dim3(p.tiles * p.Hk * (p.tile_rows / 16) * (D / 32), p.B), dim3(MERGE_THREADS), 0, st, ptb_pdl_enabled(), p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}

template <int D, bool Q8>
int launch_rows(Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    CUtensorMap mk, mv;
    const long long lines = (long long)p.n_pages * p.Hk * Geo<D, Q8>::LINES;
    if (ptb_make_tmap_bf16(&mk, k_pages, 64, lines, 64, 64, Geo<D, Q8>::LINES) || ptb_make_tmap_bf16(&mv, v_pages, 64, lines, 64, 64, Geo<D, Q8>::LINES)) return -1;
    switch (p.tile_rows) {
        case 16: return launch<D, Q8, 1>(p, mk, mv, st);
        case 32: return launch<D, Q8, 2>(p, mk, mv, st);
        default: return launch<D, Q8, 4>(p, mk, mv, st);
    }
}

int sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
    }
    return n;
}
int tile_rows_of(int rows) { return rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }

}  // namespace
}  // namespace tree
}  // namespace ptb

using namespace ptb;

// Floats of workspace that ptb_paged_attn_tree needs.
PTB_API long long ptb_paged_tree_work_floats(int T, int H, int Hk, int D) {
    if (Hk <= 0 || T <= 0) return 0;
    return (long long)tree::sm_count() * 2 * (long long)tree::partial_floats(tree::tile_rows_of(T * (H / Hk)), D);
}

// T drafted tokens of each of B requests (the latest token among them) attend to their request's cached tokens and to one another.  q: [B, T, heads] bf16 with
// pitches in elements, head h at column h * D; out [B, T, H D]; lens [B]: cached tokens before the drafted ones, node i stands in slot lens[b] + i; nodes [B]
// (null: T), rows behind them come out as zeros, as do rows that see nothing; mask [B, T]: bit j, whether the node sees node j (null: a chain).  Pages
// [n_pages, Hk, 64, D]: bf16, or e4m3 with exponents [n_pages, Hk, 64].  D is 64 or 128, T at most 64, B at most 4096.
PTB_API int ptb_paged_attn_tree(const void* q, long long q_batch, long long q_row, void* out, int B, int T, int H, int Hk, int D, const int* lens, const int* nodes, const void* mask,
                                const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, float scale, float* work,
                                int* status, cudaStream_t st) {
    if (B <= 0) return 0;
    if (T < 1 || T > tree::MAX_NODES || B > tree::MAX_B) { ptb_set_error("paged attention of trees: %d requests of %d nodes (up to %d and %d)", B, T, tree::MAX_B, tree::MAX_NODES); return -1; }
    if (Hk <= 0 || H <= 0 || H % Hk) { ptb_set_error("paged attention of trees: %d heads over %d kv heads", H, Hk); return -1; }
    if (D != 64 && D != 128) { ptb_set_error("paged attention of trees: head size %d not in {64, 128}", D); return -1; }
    if (((uintptr_t)q & 7) || q_batch % 4 || q_row % 4) { ptb_set_error("paged attention of trees: rows of q need to start on 8 bytes"); return -1; }
    if (((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15) || ((uintptr_t)k_exp & 15) || ((uintptr_t)v_exp & 15) || ((uintptr_t)work & 15)) {
        ptb_set_error("paged attention of trees: pools, exponents and the workspace need to be 16-byte aligned");
        return -1;
    }
    if (!k_exp != !v_exp) { ptb_set_error("paged attention of trees: exponents of keys and of values belong together"); return -1; }
    if (pt_stride < 1 || n_pages < 1) { ptb_set_error("paged attention of trees: no pages"); return -1; }
    tree::Params p;
    memset(&p, 0, sizeof(p));
    p.q = (const __nv_bfloat16*)q; p.q_batch = q_batch; p.q_row = q_row; p.out = (__nv_bfloat16*)out; p.lens = lens; p.nodes = nodes; p.mask = (const unsigned long long*)mask;
    p.page_table = page_table; p.pt_stride = pt_stride; p.n_pages = n_pages; p.k_exp = (const uint8_t*)k_exp; p.v_exp = (const uint8_t*)v_exp; p.work = work;
    p.B = B; p.T = T; p.H = H; p.Hk = Hk; p.G = H / Hk;
    p.tile_rows = tree::tile_rows_of(T * p.G);
    p.tiles = (T * p.G + p.tile_rows - 1) / p.tile_rows;
    p.ctas = tree::sm_count();
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = status;
    if ((long long)B * p.tiles * Hk * pt_stride > 0x7fffffffll || (long long)n_pages * Hk * 128 > 0x7fffffffll) { ptb_set_error("paged attention of trees: more pages than 31 bits count"); return -1; }
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    PTB_CUDA_OK(cudaSetDevice(dev));     // the tensor-map encoder is a driver call: bind the primary context to this thread
    if (D == 128) return k_exp ? tree::launch_rows<128, true>(p, k_pages, v_pages, st) : tree::launch_rows<128, false>(p, k_pages, v_pages, st);
    return k_exp ? tree::launch_rows<64, true>(p, k_pages, v_pages, st) : tree::launch_rows<64, false>(p, k_pages, v_pages, st);
}
