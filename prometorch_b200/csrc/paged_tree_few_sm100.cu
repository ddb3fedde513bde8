// Up to 64 rows of drafted tokens (nodes times the heads of a group) against a paged cache, on the 5th-generation tensor cores with the tokens along the lanes; see
// paged_tree.cuh.
//
// The scores of a block of 128 tokens are S^T = K Q^T: a lane of tensor memory is a token, a column a row of queries.  Of a handful of rows that leaves each of a group's
// 128 softmax threads as many scores as there are rows, where rows along the lanes would leave 128 to each of a few; and a product costs by its columns.  The second product is
// O^T += V^T P^T, its lanes the elements of the head.  Sixteen warps:
//   warp 0      brings pages: keys straight to the tile the product reads, e4m3 as they are; values too (bf16), or to a ring of raw pages (e4m3); exponents;
//   warp 1      owns tensor memory and issues the products;
//   warps 4-11  softmax, two groups of four warps that take every other block, each with scores, weights, maxima, sums and an accumulator of its own.  A thread owns a token: its
//               exponents are two numbers, its sums stay in registers until the item ends.  The rows' references lie in shared memory.  They follow the maxima only
//               where one has grown by 2^8: then, and in an item's first block, the group looks for the maxima and scales its sums and its accumulator;
//   warps 12-15 e4m3: values to fp16.  bf16: of a block with drafted tokens they clear the values that must not meet a weight (see paged_tree_sm100.cu).
//
// e4m3 keys meet queries in two e4m3 parts, q = q1 + q2: four bits and the next four are what bf16 has.  They are scaled by one power of two for all rows, so
// that the largest element lies in [2^7, 2^8); the smallest step of a part is 2^-9, 2^-17 of that.  A token's exponents scale its scores, and its weights: p' = 2^(s + e_v), of which
// the sum takes 2^-e_v.
//
// What bounds it: the cache's bytes (an SM's share of the memory brings 64 KB, a block of 128 elements in bf16, in 1.5 us; everything else takes less, side by side).
#include "paged_tree_sm100.cuh"

int ptb_make_tmap_64b(CUtensorMap* map, const void* base, long long rows, int box_rows);

namespace ptb {
namespace tree {
namespace {

constexpr int THREADS = 512, REGS_SOFTMAX = 184, REGS_OTHER = 72;        // 256 x 184 + 256 x 72 = 512 x 128
constexpr int PW = 64;                   // columns of the weights' tile: a whole line of 128 bytes for each token, whatever the number of rows

template <int D, bool Q8, int N>
struct Few {
    static constexpr int KEY = Q8 ? D : 2 * D;                         // bytes of a key
    static constexpr int Q_BYTES = N * D * 2, K_TILE = BLOCK * KEY, V_TILE = BLOCK * D * 2, RAW = BLOCK * D, P_TILE = BLOCK * PW * 2;
    static constexpr int NK = Q8 ? 3 : D == 128 ? 2 : 4, NV = Q8 ? 2 : D == 128 ? 3 : 4, NR = Q8 ? (D == 128 ? 3 : 4) : 0;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + NK * K_TILE, OFF_P = OFF_V + NV * V_TILE, OFF_R = OFF_P + 2 * P_TILE, OFF_E = OFF_R + NR * RAW;
    static constexpr int OFF_M = OFF_E + (Q8 ? 8 * 2 * BLOCK : 0);     // exponents of eight blocks, then what the softmax groups share
    static constexpr int OFF_BAR = OFF_M + 5248, OFF_PLAN = OFF_BAR + 512, TOTAL = OFF_PLAN + 1024;        // and the plan
    static_assert(TOTAL + plan_bytes(MAX_B) <= 227 * 1024, "shared memory of a CTA");
    static_assert(Q_BYTES % 1024 == 0 && K_TILE % 1024 == 0, "tiles start where the swizzle does");
};

__device__ __forceinline__ void umma_f8(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(id),
                 "r"(accumulate)
                 : "memory");
}
// K-major tile of 64-byte rows, 64-byte swizzle: eight rows 512 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_64b(uint32_t saddr) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)1 << 16) | ((uint64_t)(512 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
}
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
                   "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr)
                 : "memory");
}
// N columns of this lane, arrived.
template <int N>
__device__ __forceinline__ void columns(uint32_t taddr, uint32_t* r) {
#pragma unroll
    for (int c = 0; c < N / 16; ++c) tmem_ld16(taddr + 16 * c, r + 16 * c);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])::"memory");
}
__device__ __forceinline__ void group_sync(int g) { asm volatile("bar.sync %0, 128;" ::"r"(2 + g) : "memory"); }
// Whether any of the group's threads says so.
__device__ __forceinline__ bool group_any(int g, bool mine) {
    uint32_t any;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n bar.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}" : "=r"(any) : "r"(2 + g), "r"((uint32_t)mine) : "memory");
    return any != 0;
}
// v[r] of all lanes joined for each r < N: lane l is left with row l (and 32 + l in v[1]; of sixteen rows, with row l % 16).  v is used up.
template <int N, class Op>
__device__ __forceinline__ void join_lanes(float* v, int lane, Op op) {
    constexpr int W = N < 32 ? N : 32;
    if constexpr (N < 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], 16));
    }
#pragma unroll
    for (int s = 0; s < (N > 32 ? 2 : 1); ++s) {
#pragma unroll
        for (int o = W / 2; o > 0; o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < o; ++i) {
                const float mine = up ? v[32 * s + i + o] : v[32 * s + i], other = up ? v[32 * s + i] : v[32 * s + i + o];
                v[32 * s + i] = op(mine, __shfl_xor_sync(0xffffffffu, other, o));
            }
        }
    }
    if constexpr (N > 32) v[1] = v[32];
}

template <int D, bool Q8, int N>
__global__ void __launch_bounds__(THREADS, 1) paged_tree_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params P) {
    using S = Few<D, Q8, N>;
    constexpr int NK = S::NK, NV = S::NV, NR = Q8 ? S::NR : 1;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sq = smem, *sk = smem + S::OFF_K, *sv = smem + S::OFF_V, *sp = smem + S::OFF_P, *sr = smem + S::OFF_R, *se = smem + S::OFF_E;
    // what a softmax group shares: references less the weights' scale, scales of the accumulator, maxima or sums of its warps; what both know of an item (four of them)
    float* neg_ref = reinterpret_cast<float*>(smem + S::OFF_M);                          // [2][64]
    float* alpha_s = neg_ref + 128;                                                      // [2][64]
    float* warp_s = alpha_s + 128;                                                       // [2][4][64]
    float* factor = warp_s + 512;                                                        // [4]
    unsigned long long* seen_s = reinterpret_cast<unsigned long long*>(factor + 8);      // [4][64]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
    uint64_t *q_full = bars, *q_free = bars + 1, *s_full = bars + 2, *p_ready = bars + 4, *o_full = bars + 6;            // [1], [1], [2], [2], [2]
    uint64_t *k_full = bars + 8, *k_empty = bars + 12, *v_full = bars + 16, *v_empty = bars + 20, *v_ready = bars + 24;  // [NK], [NK], [NV], [NV], [NV]
    uint64_t *raw_full = bars + 28, *raw_empty = bars + 32;                                                              // [NR], [NR]
    unsigned long long* taint = reinterpret_cast<unsigned long long*>(bars + 36);          // [8] by item: drafted tokens whose values were cleared
    int* bad_pages = reinterpret_cast<int*>(bars + 44);                // [8] by block: bits of pages that are none of the pool's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bad_pages + 8);
    int* part = reinterpret_cast<int*>(tmem_slot + 1);                 // [16]
    volatile int* abort_flag = reinterpret_cast<volatile int*>(part + 16);
    int* starts = reinterpret_cast<int*>(smem + S::OFF_PLAN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4);
        mbar_init(q_free, 1);
        for (int g = 0; g < 2; ++g) { mbar_init(&s_full[g], 1); mbar_init(&p_ready[g], 4); mbar_init(&o_full[g], 1); }
        for (int s = 0; s < NK; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
        for (int s = 0; s < NV; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); mbar_init(&v_ready[s], 4); }
        for (int s = 0; s < NR; ++s) { mbar_init(&raw_full[s], 1); mbar_init(&raw_empty[s], 4); }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 256);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    constexpr uint32_t TM_S = 0, TM_O = 128;             // two buffers of 64 columns each
    pdl_wait();
    pdl_launch_dependents();
    plan<THREADS>(P, starts, part);
    __syncthreads();
    const int all = starts[P.B], per = units_per_cta(all, P.ctas);
    const int u0 = (int)min((long long)all, (long long)blockIdx.x * per), u1 = min(all, u0 + per);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= P.B; b += THREADS) P.starts[b] = starts[b];
    bool ok = true;
    auto wait = [&](uint64_t* bar, int turn) { return ok && (mbar_try_wait(bar, (uint32_t)(turn & 1)) || (!*abort_flag && mbar_wait(bar, (uint32_t)(turn & 1), P.status))); };

    if (warp < SOFTMAX_WARP) {
        regs_dec<REGS_OTHER>();                          // one instruction for the warp group
        if (warp == 0) {
            // -------------------------------------------------------------------------------- pages
            int n = 0;                                   // block of the run
            for (int u = u0; u < u1 && ok;) {
                const Item it = item_at(P, starts, u, u1);
                const int pages = (it.r.len + it.r.nodes + PAGE - 1) / PAGE;
                int ids = 0;                             // ids of 32 pages from page `ids_from` on
                int ids_from = -1;
                for (int j = 0; j < it.n && ok; ++j, ++n) {
                    const int p0 = 2 * (it.first + j);
                    if (ids_from < 0 || p0 - ids_from >= 32) {
                        ids_from = p0;
                        ids = p0 + lane < pages ? P.page_table[(size_t)it.b * P.pt_stride + p0 + lane] : -2;        // -2: behind the last page
                        if (ids != -2 && (ids < 0 || ids >= P.n_pages)) {
                            ids = -1;
                            if (P.status && (p0 + lane) / 2 < it.first + it.n) atomicExch(P.status, PTB_ERR_BOUNDS);
                        }
                    }
                    const int page[2] = {__shfl_sync(0xffffffffu, ids, p0 - ids_from), __shfl_sync(0xffffffffu, ids, p0 + 1 - ids_from)};
                    if (lane == 0) {
                        const int there = page[1] == -2 ? 1 : 2, sK = n % NK, sV = n % NV;
                        if (n >= NK) ok = wait(&k_empty[sK], n / NK - 1);
                        if (ok) {
                            bad_pages[n & 7] = (page[0] < 0 ? 1 : 0) | (page[1] < 0 ? 2 : 0);
                            mbar_expect_tx(&k_full[sK], there * (S::K_TILE / 2 + (Q8 ? 2 * PAGE : 0)));
                            for (int x = 0; x < there; ++x) {
                                const int head = max(page[x], 0) * P.Hk + it.kvh;        // a page that is none of the pool's: any other in its place, which no row sees
                                uint8_t* dst = sk + sK * S::K_TILE;
                                if constexpr (Q8) {
                                    tma_load_2d(dst + x * (S::K_TILE / 2), &tmK, 0, head * PAGE, &k_full[sK]);
                                    bulk_g2s(se + (n & 7) * 2 * BLOCK + x * PAGE, P.k_exp + (size_t)head * PAGE, PAGE, &k_full[sK]);
                                    bulk_g2s(se + (n & 7) * 2 * BLOCK + BLOCK + x * PAGE, P.v_exp + (size_t)head * PAGE, PAGE, &k_full[sK]);
                                } else {
                                    for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + c * (BLOCK * 128) + x * 8192, &tmK, c * 64, head * PAGE, &k_full[sK]);
                                }
                            }
                            if constexpr (Q8) {
                                const int sR = n % NR;
                                if (n >= NR) ok = wait(&raw_empty[sR], n / NR - 1);
                                if (ok) {
                                    mbar_expect_tx(&raw_full[sR], there * (S::RAW / 2));
                                    for (int x = 0; x < there; ++x)
                                        tma_load_2d(sr + sR * S::RAW + x * (S::RAW / 2), &tmV, 0, (max(page[x], 0) * P.Hk + it.kvh) * (S::RAW / 2 / 128), &raw_full[sR]);
                                }
                            } else {
                                if (n >= NV) ok = wait(&v_empty[sV], n / NV - 1);
                                if (ok) {
                                    mbar_expect_tx(&v_full[sV], there * (S::V_TILE / 2));
                                    for (int x = 0; x < there; ++x)
                                        for (int c = 0; c < D / 64; ++c)
                                            tma_load_2d(sv + sV * S::V_TILE + (x * (D / 64) + c) * 8192, &tmV, c * 64, (max(page[x], 0) * P.Hk + it.kvh) * PAGE, &v_full[sV]);
                                }
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0);
                }
                u += it.n;
            }
            if (!ok) *abort_flag = 1;
        } else if (warp == 1 && lane == 0) {
            // -------------------------------------------------------------------------------- products
            constexpr uint32_t id_s = idesc<Q8>(N, 0, 0), id_o = idesc<Q8>(PW, 1, 1);        // e4m3 has the number that fp16 has
            int base = 0, item = 0, p_turn[2] = {0, 0};  // base: block of the run that the item begins with
            for (int u = u0; u < u1 && ok; ++item) {
                const Item it = item_at(P, starts, u, u1);
                const int total = it.r.len + it.r.nodes;
                auto issue_s = [&](int j) {
                    const int n = base + j, s = n % NK;
                    ok = wait(&k_full[s], n / NK);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t d = tmem + TM_S + (uint32_t)((j & 1) * 64);
                    if constexpr (Q8) {
                        const uint64_t a0 = D == 128 ? smem_desc(smem_u32(sk + s * S::K_TILE), 16, 1024) : smem_desc_64b(smem_u32(sk + s * S::K_TILE));
                        const uint64_t b0 = D == 128 ? smem_desc(smem_u32(sq), 16, 1024) : smem_desc_64b(smem_u32(sq));
#pragma unroll
                        for (int q = 0; q < 2; ++q)          // the parts of the queries
#pragma unroll
                            for (int k = 0; k < D / 32; ++k) umma_f8(d, a0 + k * 2, b0 + (q * N * D + k * 32) / 16, id_s, (q > 0 || k > 0) ? 1u : 0u);
                    } else {
                        const uint64_t a0 = smem_desc(smem_u32(sk + s * S::K_TILE), 16, 1024), b0 = smem_desc(smem_u32(sq), 16, 1024);
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int k = 0; k < 4; ++k) umma_bf16(d, a0 + (c * (BLOCK * 128) + k * 32) / 16, b0 + (c * (N * 128) + k * 32) / 16, id_s, (c > 0 || k > 0) ? 1u : 0u);
                    }
                    umma_commit(&k_empty[s]);
                    umma_commit(&s_full[j & 1]);
                    if (j + 1 == it.n) umma_commit(q_free);
                };
                ok = wait(q_full, item);
                if (ok) issue_s(0);
                if (ok && it.n > 1) issue_s(1);
                for (int j = 0; j < it.n && ok; ++j) {
                    const int g = j & 1, n = base + j, s = n % NV, t0 = (it.first + j) * BLOCK;
                    ok = wait(&p_ready[g], p_turn[g]++);
                    if (ok) ok = wait(&v_ready[s], n / NV);
                    if (!ok) break;
                    tc_fence_after();
                    // the values' tile, 64 elements of a head 8 KB apart (of a head of 64 the upper half of the lanes gets what lies behind, which nobody reads)
                    const uint64_t a0 = smem_desc(smem_u32(sv + s * S::V_TILE), 8192, 1024), b0 = smem_desc(smem_u32(sp + g * S::P_TILE), 8192, 1024);
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (x == 0 || t0 + PAGE < total)   // the second page is there
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                umma_bf16(tmem + TM_O + (uint32_t)(g * 64), a0 + (x * (D / 64) * 8192 + k * 2048) / 16, b0 + (x * 4 + k) * (2048 / 16), id_o, (j > 1 || x > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&v_empty[s]);
                    if (j + 2 >= it.n) umma_commit(&o_full[g]);
                    if (j + 2 < it.n) issue_s(j + 2);
                }
                base += it.n;
                u += it.n;
            }
            if (!ok) *abort_flag = 1;
        }
    } else if (warp < CONVERT_WARP) {
        // ------------------------------------------------------------------------------------ softmax
        regs_inc<REGS_SOFTMAX>();
        const int g = (warp - SOFTMAX_WARP) >> 2, wg = warp & 3, tid = wg * 32 + lane;       // tid: this thread's token in a block, and its element of the head
        const uint32_t lanes = tmem + ((uint32_t)(wg * 32) << 16), ts = lanes + TM_S + (uint32_t)(g * 64), to = lanes + TM_O + (uint32_t)(g * 64);
        float *nr = neg_ref + g * 64, *al = alpha_s + g * 64, *ws = warp_s + g * 256;
        int base = 0, s_turn = 0, o_turn = 0;
        constexpr float UP = weight_up<Q8>();
        constexpr float UNSET = 1e30f;                   // less a reference that no row's score has set
        // The first group brings an item's queries to the tile, with what both groups want to know of its rows.
        auto enter = [&](const Item& it, int item) {
            const int rows = it.r.nodes * P.G;
            constexpr int EACH = N * D / 8 / 128 > 0 ? N * D / 8 / 128 : 1;  // 16-byte pieces a thread
            uint4 raw[EACH];
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int x = i * 128 + tid, r = x / (D / 8), c = x % (D / 8), node = r / P.G, head = r - node * P.G;
                raw[i] = make_uint4(0, 0, 0, 0);
                if (r < rows)
                    raw[i] = *reinterpret_cast<const uint4*>(P.q + (size_t)it.b * P.q_batch + (size_t)node * P.q_row + (size_t)(it.kvh * P.G + head) * D + c * 8);
            }
            unsigned long long seen = 0;
            if (tid < N && tid < rows) {
                const int node = tid / P.G;
                seen = (P.mask ? P.mask[(size_t)it.b * P.T + node] : (2ull << node) - 1) & (it.r.nodes < 64 ? (1ull << it.r.nodes) - 1 : ~0ull);
            }
            float f = P.scale_log2, up = 1.f;
            if constexpr (Q8) {                          // the largest magnitude of all rows to [2^7, 2^8)
                uint32_t a = 0;
#pragma unroll
                for (int i = 0; i < EACH; ++i) {
                    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) a = max(a, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
                }
                a = __reduce_max_sync(0xffffffffu, a);
                uint32_t* share = reinterpret_cast<uint32_t*>(ws);           // free between items
                if (lane == 0) share[wg] = a;
                group_sync(g);
                a = max(max(share[0], share[1]), max(share[2], share[3]));
                group_sync(g);
                const int k = min(253, max(40, (int)(a >> 7)));              // biased exponent
                up = pow2(127 + 7 - k);
                f *= pow2(k - 7 - 127);
            }
            if (item > 0) ok = wait(q_free, item - 1);   // the products of the last item have read theirs
            if (tid < N) seen_s[(item & 3) * 64 + tid] = seen;
            if (tid == 0) factor[item & 3] = f;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int x = i * 128 + tid, r = x / (D / 8), c = x % (D / 8);
                if constexpr (Q8) {
                    uint32_t w1[2], w2[2];
                    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[k]));
                        v.x *= up;
                        v.y *= up;
                        const uint32_t p1 = e4m3_pack(v.x, v.y), h = e4m3x2(p1);
                        const float2 back = __half22float2(*reinterpret_cast<const __half2*>(&h));
                        const uint32_t p2 = e4m3_pack(v.x - back.x, v.y - back.y);
                        if (k & 1) { w1[k >> 1] |= p1 << 16; w2[k >> 1] |= p2 << 16; }
                        else { w1[k >> 1] = p1; w2[k >> 1] = p2; }
                    }
                    // eight elements: half of a 16-byte piece of a row of D bytes
                    const uint32_t at = D == 128 ? r * 128 + (((c >> 1) ^ (r & 7)) * 16) + (c & 1) * 8 : r * 64 + (((c >> 1) ^ ((r >> 1) & 3)) * 16) + (c & 1) * 8;
                    if (x < N * D / 8) {
                        *reinterpret_cast<uint2*>(sq + at) = make_uint2(w1[0], w1[1]);
                        *reinterpret_cast<uint2*>(sq + N * D + at) = make_uint2(w2[0], w2[1]);
                    }
                } else if (x < N * D / 8) {
                    *reinterpret_cast<uint4*>(sq + (c / 8) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) * 16)) = raw[i];
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        };
        Item it{};
        if (u0 < u1) {
            it = item_at(P, starts, u0, u1);
            if (g == 0) enter(it, 0);
        }
        for (int u = u0, item = 0; u < u1; ++item) {
            const int len = it.r.len, total = len + it.r.nodes;
            if (tid < 64) nr[tid] = UNSET;
            group_sync(g);
            uint64_t l2[N / 2];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) l2[i] = 0;
            for (int j = g; j < it.n; j += 2) {
                const int n = base + j, t0 = (it.first + j) * BLOCK, pos = t0 + tid;
                ok = wait(&s_full[g], s_turn++);
                tc_fence_after();
                float gs = factor[item & 3], ev = 0.f, un = 1.f;
                if constexpr (Q8) {
                    // behind the last token anything may lie: within what is ever stored
                    const uint32_t ke = min(191u, max(63u, (uint32_t)se[(n & 7) * 2 * BLOCK + tid])), ve = min(191u, max(63u, (uint32_t)se[(n & 7) * 2 * BLOCK + BLOCK + tid]));
                    gs = fmaxf(gs * __uint_as_float(ke << 23), 1e-30f);      // above zero: it meets -infinity
                    ev = __uint_as_float(0x4b000000u | ve) - (8388608.f + 127.f);
                    un = __uint_as_float(0x7f000000u - (ve << 23));
                }
                const bool bad = (bad_pages[n & 7] >> (tid >> 6)) & 1;
                const unsigned long long* seen = seen_s + (item & 3) * 64;
                uint32_t r[N];
                auto scores = [&] {
                    columns<N>(ts, r);
                    if (bad || pos >= total) {
#pragma unroll
                        for (int i = 0; i < N; ++i) r[i] = 0xff800000u;      // -infinity
                    } else if (pos >= len) {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            if (!((seen[i] >> (pos - len)) & 1)) r[i] = 0xff800000u;
                    }
                };
                // x = score - reference, in powers of two
                const uint64_t g2 = both(gs), e2 = both(ev);
                auto relate = [&] {
#pragma unroll
                    for (int i = 0; i < N; i += 4) {
                        const float4 m = *reinterpret_cast<const float4*>(nr + i);
                        uint64_t a = pair(__float_as_uint(m.x), __float_as_uint(m.y)), b = pair(__float_as_uint(m.z), __float_as_uint(m.w));
                        if constexpr (Q8) { a = add2(a, e2); b = add2(b, e2); }
                        float x[4];
                        apart(fma2(pair(r[i], r[i + 1]), g2, a), x[0], x[1]);
                        apart(fma2(pair(r[i + 2], r[i + 3]), g2, b), x[2], x[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) r[i + k] = __float_as_uint(x[k]);
                    }
                };
                scores();
                relate();
                float m4[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < N; i += 2) m4[(i >> 1) & 1] = max3(m4[(i >> 1) & 1], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                if (group_any(g, fmaxf(m4[0], m4[1]) > 8.f + UP)) {          // a maximum that has grown by 2^8, or that is not known yet
                    scores();
                    float v[N];
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] = fmaf(__uint_as_float(r[i]), gs, ev);
                    join_lanes<N>(v, lane, [](float a, float b) { return fmaxf(a, b); });
                    if (lane < N) ws[wg * 64 + lane] = v[0];
                    if (N > 32) ws[wg * 64 + 32 + lane] = v[1];
                    group_sync(g);
                    if (tid < N) {
                        const float mx = fmaxf(fmaxf(ws[tid], ws[64 + tid]), fmaxf(ws[128 + tid], ws[192 + tid])), old = nr[tid];
                        float a = 1.f;
                        if (mx + old > 8.f + UP) {
                            a = old == UNSET ? 0.f : exp2f(-mx + UP - old);
                            nr[tid] = UP - mx;
                        }
                        al[tid] = a;
                    }
                    group_sync(g);
                    const bool scale = j > 1 && (D == 128 || wg < 2);
                    if (scale) {                         // these scores are there, so the product before them is done
                        uint32_t o[N];
                        columns<N>(to, o);
#pragma unroll
                        for (int i = 0; i < N; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al[i]);
#pragma unroll
                        for (int c = 0; c < N / 16; ++c) tmem_st16(to + 16 * c, o + 16 * c);
                        tmem_st_wait();
                    }
#pragma unroll
                    for (int i = 0; i < N / 2; ++i) {
                        float a, b;
                        apart(l2[i], a, b);
                        l2[i] = pair(__float_as_uint(a * al[2 * i]), __float_as_uint(b * al[2 * i + 1]));
                    }
                    scores();
                    relate();
                }
                uint8_t* pt = sp + g * S::P_TILE + tid * 128;
                const uint64_t un2 = both(un);
#pragma unroll
                for (int c = 0; c < N / 8; ++c) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int i = 8 * c + 2 * k;
                        const float x = exp2f(__uint_as_float(r[i])), y = exp2f(__uint_as_float(r[i + 1]));
                        const uint64_t xy = pair(__float_as_uint(x), __float_as_uint(y));
                        if constexpr (Q8) l2[i / 2] = fma2(xy, un2, l2[i / 2]);
                        else l2[i / 2] = add2(l2[i / 2], xy);
                        w[k] = pack2<Q8>(x, y);
                    }
                    *reinterpret_cast<uint4*>(pt + ((c ^ (tid & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                }
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[g]);
            }
            // ---- the item's part of this group; the next item's scores are computed meanwhile
            const Item next = u + it.n < u1 ? item_at(P, starts, u + it.n, u1) : it;
            if (g == 0 && u + it.n < u1) enter(next, item + 1);
            // Of an item that no other CTA has a part of, the groups join their parts here, each for half of the rows.
            const bool whole = it.n == it.r.units, shared = whole && it.n > 1;
            float* wk = P.work + partial_at(P, blockIdx.x, u == u0 ? 0 : 1, g, D);
            float2* ml = reinterpret_cast<float2*>(wk + (size_t)N * D);
            const int rows = min(N, it.r.nodes * P.G);
            float v[N];
#pragma unroll
            for (int i = 0; i < N / 2; ++i) apart(l2[i], v[2 * i], v[2 * i + 1]);
            join_lanes<N>(v, lane, [](float a, float b) { return a + b; });
            group_sync(g);                               // the maxima have been read
            if (lane < N) ws[wg * 64 + lane] = v[0];
            if (N > 32) ws[wg * 64 + 32 + lane] = v[1];
            group_sync(g);
            float2 mine = make_float2(-INFINITY, 0.f);
            if (tid < rows && nr[tid] != UNSET) mine = make_float2(UP - nr[tid], (ws[tid] + ws[64 + tid]) + (ws[128 + tid] + ws[192 + tid]));
            if (tid < rows) ml[tid] = mine;
            if (it.n > g) ok = wait(&o_full[g], o_turn++);
            tc_fence_after();
            uint32_t o[N];
            if (it.n > g && (D == 128 || wg < 2)) {
                columns<N>(to, o);
                for (unsigned long long left = taint[item & 7]; left; left &= left - 1) {        // values that were cleared: for the rows that see their token
                    const int d = __ffsll((long long)left) - 1, t = len + d;
                    if (t / BLOCK < it.first || t / BLOCK >= it.first + it.n || ((t / BLOCK - it.first) & 1) != g) continue;
                    const int page = P.page_table[(size_t)it.b * P.pt_stride + t / PAGE];
                    if (page < 0 || page >= P.n_pages) continue;
                    const size_t v_at = (((size_t)page * P.Hk + it.kvh) * PAGE + t % PAGE) * D + tid;
                    const uint32_t w = Q8 ? 0x7fffffffu : (uint32_t)reinterpret_cast<const uint16_t*>(P.v_raw)[v_at] << 16;
                    if (Q8 ? (P.v_raw[v_at] & 0x7f) == 0x7f : (w & 0x7f800000u) == 0x7f800000u) {
#pragma unroll
                        for (int i = 0; i < N; ++i)
                            if ((seen_s[(item & 3) * 64 + i] >> d) & 1) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(w));
                    }
                }
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (i < rows && (!whole || (shared && (i < N / 2) == (g == 1)))) wk[(size_t)i * D + tid] = __uint_as_float(o[i]);
            }
            if (whole) {
                if (shared) both_sync();
                const float2* ml1 = reinterpret_cast<const float2*>(wk + (g ? -1 : 1) * (long long)partial_floats(N, D) + (size_t)N * D);
                if (tid < N) {
                    const float2 other = shared && tid < rows ? ml1[tid] : make_float2(-INFINITY, 0.f);
                    const float top = fmaxf(mine.x, other.x), a = mine.x == -INFINITY ? 0.f : exp2f(mine.x - top), b = other.x == -INFINITY ? 0.f : exp2f(other.x - top);
                    const float sum = mine.y * a + other.y * b, inv = sum != 0.f ? 1.f / sum : 0.f;
                    al[tid] = a * inv;
                    ws[tid] = b * inv;
                }
                group_sync(g);
                if (it.n > g && (D == 128 || wg < 2)) {
                    const float* theirs = wk + (g ? -1 : 1) * (long long)partial_floats(N, D);
                    __nv_bfloat16* out = P.out + ((size_t)it.b * P.T * P.H + it.kvh * P.G) * D + tid;
                    int head = 0;                        // of row i: out is at head 0 of its node
#pragma unroll
                    for (int i = 0; i < N; ++i) {
                        if (i < ((rows + 15) & ~15) && i < P.T * P.G && (!shared || (i < N / 2) == (g == 0))) {      // sixteen rows at a time, the ones behind the last are zeros
                            const float a = al[i], b = shared ? ws[i] : 0.f;
                            float y = 0.f;
                            if (a != 0.f) y = __uint_as_float(o[i]) * a;
                            if (b != 0.f) y += theirs[(size_t)i * D + tid] * b;
                            out[(size_t)head * D] = __float2bfloat16_rn(i < rows ? y : 0.f);
                        }
                        if (++head == P.G) { head = 0; out += (size_t)P.H * D; }
                    }
                }
            }
            tc_fence_before();
            base += it.n;
            u += it.n;
            it = next;
            both_sync();                                 // references and sums have been read; and neither group is more than an item ahead of the other
        }
        if (!ok) *abort_flag = 1;
    } else {
        // ------------------------------------------------------------------------------------ values
        regs_dec<REGS_OTHER>();
        const int cw = warp - CONVERT_WARP, tid = threadIdx.x - CONVERT_WARP * 32;
        int n = 0, item = 0;
        for (int u = u0; u < u1; ++item) {               // after a wait that ran out as well: the four warps meet at every item
            const Item it = item_at(P, starts, u, u1);
            const int len = it.r.len, total = len + it.r.nodes;
            if (tid == 0) taint[item & 7] = 0;           // eight items back: nobody reads it any more
            convert_sync();
            for (int j = 0; j < it.n; ++j, ++n) {
                const int t0 = (it.first + j) * BLOCK, sV = n % NV;
                if constexpr (!Q8) {
                    ok = wait(&v_full[sV], n / NV);
                    const int t = t0 + tid;
                    if (ok && t0 + BLOCK > len && t >= len) {
                        uint8_t* v = sv + sV * S::V_TILE + (tid >> 6) * (D / 64) * 8192 + (tid & 63) * 128;
                        bool odd = false;
                        for (int i = 0; i < D / 8; ++i) {
                            uint4* w = reinterpret_cast<uint4*>(v + (i / 8) * 8192 + (i & 7) * 16);
                            if (t >= total) { *w = make_uint4(0, 0, 0, 0); continue; }
                            uint4 x = *w;
                            uint32_t* y = reinterpret_cast<uint32_t*>(&x);
                            uint32_t any = 0;
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t no = __vcmpeq2(y[k] & 0x7f807f80u, 0x7f807f80u);
                                any |= no;
                                y[k] &= ~no;
                            }
                            if (any) { *w = x; odd = true; }
                        }
                        if (odd) atomicOr(&taint[item & 7], 1ull << (t - len));
                    }
                } else {
                    // A warp takes 32 tokens, eight of them and 64 of their elements at a time: lane (token, 16-byte piece).  Two tokens of a phase differ in the bits that part their
                    // pieces in the raw lines and in the tile's, so that neither meets in a bank; all offsets but this lane's are constants
                    constexpr int HALVES = D / 64;
                    const int sR = n % NR, pr = lane >> 3, sel = (lane >> 2) & 1, c4 = lane & 3, in8 = D == 128 ? (sel ? pr ^ 5 : pr) : 2 * pr + sel;
                    const uint32_t from = D == 128 ? cw * 4096 + in8 * 128 + ((c4 ^ in8) * 16) : cw * 2048 + (in8 >> 1) * 128 + ((((in8 & 1) * 4 + c4) ^ (in8 >> 1)) * 16);
                    const uint32_t to = (cw & 1) * 4096 + (cw >> 1) * HALVES * 8192 + in8 * 128 + (((2 * c4) ^ in8) * 16);
                    auto convert = [&](auto some_) {
                        constexpr bool SOME = decltype(some_)::value;        // a block with drafted tokens
                        const uint8_t* raw = sr + sR * S::RAW;
                        uint8_t* tile = sv + sV * S::V_TILE;
                        uint4 w[4 * HALVES];
#pragma unroll
                        for (int i = 0; i < 4 * HALVES; ++i) w[i] = *reinterpret_cast<const uint4*>(raw + (D == 128 ? (from + i / HALVES * 1024) ^ (i % HALVES * 64) : (from + i * 512) ^ ((i & 1) * 64)));
#pragma unroll
                        for (int i = 0; i < 4 * HALVES; ++i) {
                            uint32_t y[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                            if constexpr (SOME) {                            // what lies behind the last token, and what is no number of a drafted one
                                const int token = t0 + cw * 32 + i / HALVES * 8 + in8;
                                uint32_t any = 0;
#pragma unroll
                                for (int k = 0; k < 4; ++k) {
                                    const uint32_t no = token >= total ? ~0u : token >= len ? __vcmpeq4(y[k] & 0x7f7f7f7fu, 0x7f7f7f7fu) : 0u;
                                    any |= no;
                                    y[k] &= ~no;
                                }
                                if (any && token < total) atomicOr(&taint[item & 7], 1ull << (token - len));
                            }
                            uint32_t h[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) h[k] = e4m3x2(k & 1 ? y[k >> 1] >> 16 : y[k >> 1]);
                            const uint32_t at = i / HALVES * 1024 + i % HALVES * 8192;
                            *reinterpret_cast<uint4*>(tile + to + at) = make_uint4(h[0], h[1], h[2], h[3]);
                            *reinterpret_cast<uint4*>(tile + (to ^ 16) + at) = make_uint4(h[4], h[5], h[6], h[7]);
                        }
                    };
                    ok = wait(&raw_full[sR], n / NR);
                    if (ok && n >= NV) ok = wait(&v_empty[sV], n / NV - 1);
                    if (ok && t0 + BLOCK <= len) convert(Flag<false>());
                    else if (ok) convert(Flag<true>());
                    if (lane == 0) mbar_arrive(&raw_empty[sR]);
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_ready[sV]);
                ok = __all_sync(0xffffffffu, ok);
            }
            u += it.n;
        }
        if (!ok) *abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, 256);
}

template <int D, bool Q8, int N>
int launch_n(const Params& p, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t st) {
    using S = Few<D, Q8, N>;
    static bool attr[64];
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        PTB_CUDA_OK(cudaFuncSetAttribute(paged_tree_few_kernel<D, Q8, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL + plan_bytes(MAX_B)));
        if (dev < 64) attr[dev] = true;
    }
    PTB_CUDA_OK(ptb_launch(paged_tree_few_kernel<D, Q8, N>, dim3(p.ctas), dim3(THREADS), (size_t)S::TOTAL + plan_bytes(p.B), st, ptb_pdl_enabled(), mk, mv, p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}

}  // namespace

// All items' partial results, two for each CTA and item; tile_rows is 16, 32 or 64.
template <int D, bool Q8>
int launch_few(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    CUtensorMap mk, mv;
    const long long rows = (long long)p.n_pages * p.Hk * PAGE;
    if constexpr (Q8) {                                  // keys: rows of a token; values: 128-byte lines of raw pages
        if (D == 128 ? ptb_make_tmap_bf16(&mk, k_pages, 64, rows, 64, 64, PAGE) : ptb_make_tmap_64b(&mk, k_pages, rows, PAGE)) return -1;
        if (ptb_make_tmap_bf16(&mv, v_pages, 64, rows * D / 128, 64, 64, PAGE * D / 128)) return -1;
    } else {
        if (ptb_make_tmap_bf16(&mk, k_pages, D, rows, D, 64, PAGE) || ptb_make_tmap_bf16(&mv, v_pages, D, rows, D, 64, PAGE)) return -1;
    }
    switch (p.tile_rows) {
        case 16: return launch_n<D, Q8, 16>(p, mk, mv, st);
        case 32: return launch_n<D, Q8, 32>(p, mk, mv, st);
        default: return launch_n<D, Q8, 64>(p, mk, mv, st);
    }
}
template int launch_few<64, false>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<64, true>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<128, false>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<128, true>(const Params&, const void*, const void*, cudaStream_t);

}  // namespace tree
}  // namespace ptb
