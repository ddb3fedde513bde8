// Drafted tokens against a paged cache on the 5th-generation tensor cores with the tokens along the lanes, up to 64 rows (nodes times the heads of a group) at a time; see paged_tree.cuh.
//
// The scores of a block of 128 tokens are S^T = K Q^T: a lane of tensor memory is a token, a column a row of queries.  Of a handful of rows that leaves each of a group's
// 128 softmax threads as many scores as there are rows, where rows along the lanes would leave 128 to each of a few; and a product costs by its columns.  The second product is
// O^T += V^T P^T, its lanes the elements of the head.  Sixteen warps:
//   warp 0      brings pages, keys and values straight to the tiles that the products read, and exponents;
//   warp 1      owns tensor memory and issues the products;
//   warps 4-11  softmax, two groups of four warps.  A thread owns a token: its exponents are two numbers, its sums stay in registers until the item ends.  The rows' references lie
//               in shared memory.  They follow the maxima only where one has grown by 2^GROW: then, and in an item's first block, a group looks for the maxima and
//               scales its sums and its accumulator.  Up to 32 rows the groups take every other block, each with references, sums and an accumulator of its own, so that a
//               block's chain of waits lasts two blocks' time; of more rows, for which one thread has not the registers, each group takes half of them in every block;
//   warps 12-15 bring an item's queries, with what the softmax wants to know of its rows, while the item before it is at work; and of a block with drafted tokens
//               they clear the values that must not meet a weight (see paged_tree_sm100.cu).
//
// e4m3: both products have 8-bit operands, and nothing is converted but what the kernel makes itself.  Queries become two e4m3 parts, q = q1 + q2: four bits and the next four
// are what bf16 has; a row is scaled by a power of two, so that its largest element lies in [2^7, 2^8), the smallest step of a part is 2^-9, 2^-17 of that.  A token's
// exponents scale its scores, and its weights: p' = 2^(s + e_v), of which the sum takes 2^-e_v (exponents of a row's values may be 100 apart: the sum of those with the least then still
// has its place below one with the largest; zeros have the least there is, -64).  Weights are rounded to fp16, and become three e5m2 parts, which are top bytes of fp16: a part to nearest
// leaves at most an eighth of its power of two, with a sign, so that p = p1 + p2 + p3 has all eleven bits.  The parts' smallest step is 2^-16: at most 2^-17, 2^-28 of an item's largest
// weights, is lost of a small one.  Parts are columns of their own, of scores and of accumulators, so that a page is read once.
//
// bf16: weights become two bf16 parts, themselves rounded and what that leaves, columns of their own as well; at most 2^-16 of a weight is lost.
//
// What bounds it.  Shared memory takes 128 bytes a cycle, and a product of few columns costs what its 4 KB of keys or values take (measured 42 cycles alone).  bf16: pages 64 KB written and
// 64 KB read, weights (two parts) and queries 40 KB (64 rows: 80): 1340 (1660) cycles a block of 128 elements, of the 2100
// that the SM's share of the memory takes.  e4m3: 32 + 32 KB, and 32 KB for the parts, 750 cycles of 1050.  Measured are 1300 with 16 rows (the chain of waits of the warp that issues the products), 1500 with 32 and 2400 with 64 (the softmax's): e4m3, 32 requests of 8192 tokens,
// 4 rows, 84 us, 74 % of the copy rate.  Values converted to fp16, the fp16 product and the two parts of queries one after the other took 148.
#include "paged_tree_sm100.cuh"

int ptb_make_tmap_64b(CUtensorMap* map, const void* base, long long rows, int box_rows);

namespace ptb {
namespace tree {
namespace {

constexpr int THREADS = 512, REGS_SOFTMAX = 184, REGS_OTHER = 72;        // 256 x 184 + 256 x 72 = 512 x 128
template <int D, bool Q8, int N>
struct Few {
    static constexpr int KEY = Q8 ? D : 2 * D;                         // bytes of a key, or a value
    static constexpr int Q_PARTS = Q8 ? 2 : 1, P_PARTS = Q8 ? 3 : 2;
    static constexpr int Q_BYTES = N * D * 2, TILE = BLOCK * KEY;
    static constexpr int S_COLS = Q_PARTS * N;                         // columns of scores
    static constexpr int O_COLS = P_PARTS * N;                         // of an accumulator, and of the weights' tile
    static constexpr int P_TILE = BLOCK * (N == 64 ? 256 : 128);       // lines of 128 bytes
    static constexpr int TMEM = Q8 ? 512 : 256, TM_O = 2 * (Q8 ? 128 : 64);
    static constexpr int NK = KEY == 256 ? 2 : KEY == 128 && N == 64 ? 4 : 5, NV = KEY == 256 ? (N == 64 ? 2 : 3) : NK;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + NK * TILE, OFF_P = OFF_V + NV * TILE, OFF_E = OFF_P + 2 * P_TILE;
    static constexpr int OFF_M = OFF_E + (Q8 ? 8 * 2 * BLOCK : 0);     // exponents of eight blocks, then what the softmax groups share
    static constexpr int OFF_BAR = OFF_M + 5120 + 1024, OFF_PLAN = OFF_BAR + 512, TOTAL = OFF_PLAN + 1024;         // and the plan
    static_assert(TOTAL + plan_bytes(MAX_B) <= 227 * 1024, "shared memory of a CTA");
    static_assert(Q_BYTES % 1024 == 0 && TILE % 1024 == 0, "tiles start where the swizzle does");
    static_assert(NK <= 5, "blocks whose scores are being weighed and those on their way are fewer than eight");
};

// Products, of which the whole warp knows the operands and one lane (`lead`) issues them: in a branch of that lane alone each would gather its operands anew.
__device__ __forceinline__ uint32_t elect_lead() {
    uint32_t lead;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(lead));
    return lead;
}
template <bool F8>
__device__ __forceinline__ void product(uint32_t lead, uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t id, uint32_t accumulate) {
    if constexpr (F8)
        asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d), "l"(desc_a),
                     "l"(desc_b), "r"(id), "r"(accumulate), "r"(lead)
                     : "memory");
    else
        asm volatile("{\n .reg .pred p, q;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(tmem_d), "l"(desc_a),
                     "l"(desc_b), "r"(id), "r"(accumulate), "r"(lead)
                     : "memory");
}
// Rows of 64 bytes, 64-byte swizzle: eight of them 512 bytes apart.
__device__ __forceinline__ uint64_t smem_desc_64b(uint32_t saddr, uint32_t lbo) {
    return (uint64_t)((saddr >> 4) & 0x3FFF) | ((uint64_t)(lbo >> 4) << 16) | ((uint64_t)(512 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)4 << 61);
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
// v[r] of all lanes joined for each r < N: v[0] is row lane % N in the end.  The others are used up.
template <int N, class Op>
__device__ __forceinline__ void join_lanes(float* v, int lane, Op op) {
    if constexpr (N < 32) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = op(v[i], __shfl_xor_sync(0xffffffffu, v[i], 16));
    }
#pragma unroll
    for (int o = N / 2; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int i = 0; i < o; ++i) {
            const float mine = up ? v[i + o] : v[i], other = up ? v[i] : v[i + o];
            v[i] = op(mine, __shfl_xor_sync(0xffffffffu, other, o));
        }
    }
}

// Two fp16 whose top bytes are e5m2 numbers next to them, and what those leave, exactly.
__device__ __forceinline__ uint32_t top_bytes(uint32_t w) { return w + 0x00800080u; }
__device__ __forceinline__ uint32_t less_top_bytes(uint32_t w, uint32_t near) {
    const uint32_t top = near & 0xff00ff00u;
    const __half2 d = __hsub2(*reinterpret_cast<const __half2*>(&w), *reinterpret_cast<const __half2*>(&top));
    return *reinterpret_cast<const uint32_t*>(&d);
}

template <int D, bool Q8, int N>
__global__ void __launch_bounds__(THREADS, 1) paged_tree_few_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params P) {
    using S = Few<D, Q8, N>;
    constexpr int NK = S::NK, NV = S::NV;
    constexpr bool SPLIT = N == 64;                      // the groups part the rows, not the blocks
    constexpr int R = SPLIT ? 32 : N;                    // rows of a softmax thread
    auto tile_row = [](const Item& it) { return N == 64 ? it.tile * N : 0; };        // an item's first row: of fewer than 64 there is one tile
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sq = smem, *sk = smem + S::OFF_K, *sv = smem + S::OFF_V, *sp = smem + S::OFF_P, *se = smem + S::OFF_E;
    // what a softmax group shares: the weights' scale less the references, scales of the accumulator, maxima or sums of its warps; what both know of an item (four of them)
    float* neg_ref = reinterpret_cast<float*>(smem + S::OFF_M);                          // [2][64]
    float* alpha_s = neg_ref + 128;                                                      // [2][64]
    float* warp_s = alpha_s + 128;                                                       // [2][4][64]
    float* factor = warp_s + 512;                                                        // [4][64] e4m3
    unsigned long long* seen_s = reinterpret_cast<unsigned long long*>(factor + 256);    // [4][64]
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
    uint64_t *q_full = bars, *q_free = bars + 1, *s_full = bars + 2, *p_ready = bars + 4, *o_full = bars + 6;            // [1], [1], [2], [2], [2]
    uint64_t *k_full = bars + 8, *k_empty = bars + 14, *v_full = bars + 20, *v_empty = bars + 26, *v_ready = bars + 32;  // [NK], [NK], [NV], [NV], [NV]
    unsigned long long* taint = reinterpret_cast<unsigned long long*>(bars + 38);          // [8] by item: drafted tokens whose values were cleared
    int* bad_pages = reinterpret_cast<int*>(bars + 46);                // [8] by block: bits of pages that are none of the pool's
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bad_pages + 8);
    int* part = reinterpret_cast<int*>(tmem_slot + 1);                 // [16]
    volatile int* abort_flag = reinterpret_cast<volatile int*>(part + 16);
    int* starts = reinterpret_cast<int*>(smem + S::OFF_PLAN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        mbar_init(q_full, 4);
        mbar_init(q_free, 1);
        for (int g = 0; g < 2; ++g) { mbar_init(&s_full[g], 1); mbar_init(&p_ready[g], SPLIT ? 8 : 4); mbar_init(&o_full[g], 1); }
        for (int s = 0; s < NK; ++s) { mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1); }
        for (int s = 0; s < NV; ++s) { mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1); mbar_init(&v_ready[s], 4); }
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, S::TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    constexpr uint32_t TM_S = 0, TM_O = S::TM_O;         // two buffers of scores, two accumulators (64 rows: one)
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
            int n = 0, sent_v = 0;                       // block of the run; blocks whose values are on their way or there
            if (u0 < u1) asm volatile("bar.sync 5, 160;" ::: "memory");          // the first queries go before the first pages, behind which they would wait
            for (int u = u0; u < u1 && ok;) {
                const Item it = item_at(P, starts, u, u1);
                const int pages = (it.r.len + it.r.nodes + PAGE - 1) / PAGE;
                int ids = 0;                             // ids of 32 pages from page `ids_from` on
                int ids_from = -1;
                for (int j = 0; j < it.n && ok; ++j, ++n) {
                    const int p0 = 2 * (it.first + j);
                    if (ids_from < 0 || p0 - ids_from >= 32) {
                        ids_from = p0;
                        ids = p0 + lane < pages ? P.page_table[(size_t)it.b * P.pt_stride + p0 + lane] : 0;
                        if (ids < 0 || ids >= P.n_pages) {
                            ids = -1;
                            if (P.status && (p0 + lane) / 2 < it.first + it.n) atomicExch(P.status, PTB_ERR_BOUNDS);
                        }
                    }
                    const int page[2] = {__shfl_sync(0xffffffffu, ids, p0 - ids_from), __shfl_sync(0xffffffffu, ids, p0 + 1 - ids_from)};
                    if (lane == 0) {
                        const int there = p0 + 1 < pages ? 2 : 1, sK = n % NK, sV = n % NV;
                        if (n >= NK) ok = wait(&k_empty[sK], n / NK - 1);
                        else if (n >= 2) ok = wait(&k_full[n - 2], 0);               // two blocks under way at a time: what others fetch does not wait behind a whole ring
                        if (ok) {
                            bad_pages[n & 7] = (page[0] < 0 ? 1 : 0) | (page[1] < 0 ? 2 : 0);
                            mbar_expect_tx(&k_full[sK], there * (S::TILE / 2 + (Q8 ? 2 * PAGE : 0)));
                            auto page_to = [&](uint8_t* dst, const CUtensorMap* map, int x, uint64_t* bar) {         // a page that is none of the pool's: any other in its place, which no row sees and whose values are cleared
                                const int row = (max(page[x], 0) * P.Hk + it.kvh) * PAGE;
                                if constexpr (Q8) tma_load_2d(dst + x * (S::TILE / 2), map, 0, row, bar);
                                else
                                    for (int c = 0; c < D / 64; ++c) tma_load_2d(dst + (map == &tmK ? c * (BLOCK * 128) + x * 8192 : (x * (D / 64) + c) * 8192), map, c * 64, row, bar);
                            };
                            for (int x = 0; x < there; ++x) {
                                page_to(sk + sK * S::TILE, &tmK, x, &k_full[sK]);
                                if constexpr (Q8) {
                                    const size_t exps = (size_t)(max(page[x], 0) * P.Hk + it.kvh) * PAGE;
                                    bulk_g2s(se + (n & 7) * 2 * BLOCK + x * PAGE, P.k_exp + exps, PAGE, &k_full[sK]);
                                    bulk_g2s(se + (n & 7) * 2 * BLOCK + BLOCK + x * PAGE, P.v_exp + exps, PAGE, &k_full[sK]);
                                }
                            }
                            if (n >= NV) ok = wait(&v_empty[sV], n / NV - 1);
                            if (ok) {
                                mbar_expect_tx(&v_full[sV], there * (S::TILE / 2));
                                for (int x = 0; x < there; ++x) page_to(sv + sV * S::TILE, &tmV, x, &v_full[sV]);
                                sent_v = n + 1;
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, (int)ok, 0);
                }
                u += it.n;
            }
            if (!ok) {
                *abort_flag = 1;
                if (lane == 0) drain<NK, NV>(k_full, v_full, n, sent_v, P.status);
            }
        } else if (warp == 1) {
            // -------------------------------------------------------------------------------- products
            constexpr uint32_t id_s = idesc<Q8>(S::S_COLS, 0, 0);                            // e4m3 has the number that fp16 has
            constexpr uint32_t id_o = idesc<Q8>(S::O_COLS, 1, 1) | (Q8 ? 1u << 10 : 0u);     // e5m2 weights
            const uint32_t lead = elect_lead();
            const uint64_t q0 = Q8 && D == 64 ? smem_desc_64b(smem_u32(sq), 16) : smem_desc(smem_u32(sq), 16, 1024);
            int base = 0, item = 0, p_turn[2] = {0, 0};  // base: block of the run that the item begins with
            for (int u = u0; u < u1 && ok; ++item) {
                const Item it = item_at(P, starts, u, u1);
                const int total = it.r.len + it.r.nodes;
                auto issue_s = [&](int j) {
                    const int n = base + j, s = n % NK;
                    ok = wait(&k_full[s], n / NK);
                    if (!ok) return;
                    tc_fence_after();
                    const uint32_t d = tmem + TM_S + (uint32_t)((j & 1) * (TM_O / 2));
                    const uint64_t k0 = Q8 && D == 64 ? smem_desc_64b(smem_u32(sk + s * S::TILE), 16) : smem_desc(smem_u32(sk + s * S::TILE), 16, 1024);
                    if constexpr (Q8) {
#pragma unroll
                        for (int k = 0; k < D / 32; ++k) product<true>(lead, d, k0 + k * 2, q0 + k * 2, id_s, k > 0 ? 1u : 0u);
                    } else {
#pragma unroll
                        for (int c = 0; c < D / 64; ++c)
#pragma unroll
                            for (int k = 0; k < 4; ++k)
                                product<false>(lead, d, k0 + (c * (BLOCK * 128) + k * 32) / 16, q0 + (c * (N * 128) + k * 32) / 16, id_s, (c > 0 || k > 0) ? 1u : 0u);
                    }
                    if (lead) {
                        umma_commit(&s_full[j & 1]);
                        umma_commit(&k_empty[s]);
                        if (j + 1 == it.n) umma_commit(q_free);
                    }
                    __syncwarp();
                };
                ok = wait(q_full, item);
                if (ok) issue_s(0);
                if (ok && it.n > 1) issue_s(1);
                for (int j = 0; j < it.n && ok; ++j) {
                    const int g = j & 1, n = base + j, s = n % NV, t0 = (it.first + j) * BLOCK;
                    ok = wait(&v_ready[s], n / NV);
                    if (ok) ok = wait(&p_ready[g], p_turn[g]++);
                    if (!ok) break;
                    tc_fence_after();
                    const uint64_t p0 = smem_desc(smem_u32(sp + g * S::P_TILE), BLOCK * 128, 1024);
                    const uint32_t d = tmem + TM_O + (uint32_t)(SPLIT ? 0 : g * S::O_COLS);
                    // of a head of 64 the upper half of the lanes gets what lies 8 KB behind, which nobody reads
                    const uint64_t v0 = Q8 && D == 64 ? smem_desc_64b(smem_u32(sv + s * S::TILE), 8192) : smem_desc(smem_u32(sv + s * S::TILE), 8192, 1024);
                    constexpr int STEP = Q8 ? 32 : 16, STEPS = PAGE / STEP;  // tokens of a product, products of a page
#pragma unroll
                    for (int x = 0; x < 2; ++x)
                        if (x == 0 || t0 + PAGE < total)   // the second page is there
#pragma unroll
                            for (int k = 0; k < STEPS; ++k)
                                product<Q8>(lead, d, v0 + (x * (S::TILE / 2) + k * STEP * (Q8 ? D : 128)) / 16, p0 + (x * STEPS + k) * (STEP * 128 / 16), id_o,
                                            (j > (SPLIT ? 0 : 1) || x > 0 || k > 0) ? 1u : 0u);
                    if (lead) {
                        umma_commit(&v_empty[s]);
                        if (SPLIT ? j + 1 == it.n : j + 2 >= it.n) umma_commit(&o_full[SPLIT ? 0 : g]);
                    }
                    __syncwarp();
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
        const int r0 = SPLIT ? g * R : 0;                // the group's first row
        const uint32_t lanes = tmem + ((uint32_t)(wg * 32) << 16), to = lanes + TM_O + (uint32_t)(SPLIT ? r0 : g * S::O_COLS);
        float *nr = neg_ref + g * 64, *al = alpha_s + g * 64, *ws = warp_s + g * 256;
        int base = 0, s_turn = 0, o_turn = 0;            // s_turn: a bit for each buffer
        constexpr float UP = Q8 ? 11.f : 0.f, GROW = Q8 ? 4.f : 8.f;         // the largest weight is 2^(UP + GROW): e5m2 ends below 2^16
        constexpr float UNSET = 1e30f;                   // a row that has seen nothing: whatever it sees outgrows this
        Item it{};
        if (u0 < u1) it = item_at(P, starts, u0, u1);
        for (int u = u0, item = 0; u < u1; ++item) {
            const int len = it.r.len, total = len + it.r.nodes;
            if (tid < 64) nr[tid] = 0.f;
            bool known = false;                          // of row tid: it has a reference
            group_sync(g);
            const bool some = SPLIT || it.n > g;         // this group has blocks
            uint64_t l2[R / 2];
#pragma unroll
            for (int i = 0; i < R / 2; ++i) l2[i] = 0;
            for (int j = SPLIT ? 0 : g; j < it.n; j += SPLIT ? 1 : 2) {
                const int n = base + j, t0 = (it.first + j) * BLOCK, pos = t0 + tid, buf = j & 1;
                const uint32_t ts = lanes + TM_S + (uint32_t)(buf * (TM_O / 2) + r0);
                ok = wait(&s_full[buf], s_turn >> buf);
                s_turn ^= 1 << buf;
                tc_fence_after();
                float gs = P.scale_log2, ev = 0.f, un = 1.f;
                if constexpr (Q8) {
                    // behind the last token anything may lie: within what is ever stored
                    const uint32_t ke = min(191u, max(63u, (uint32_t)se[(n & 7) * 2 * BLOCK + tid])), ve = min(191u, max(63u, (uint32_t)se[(n & 7) * 2 * BLOCK + BLOCK + tid]));
                    gs = __uint_as_float(ke << 23);
                    ev = __uint_as_float(0x4b000000u | ve) - (8388608.f + 127.f);
                    un = __uint_as_float(0x7f000000u - (ve << 23));
                }
                const bool bad = (bad_pages[n & 7] >> (tid >> 6)) & 1;
                const unsigned long long* seen = seen_s + (item & 3) * 64 + r0;
                const float* fac = factor + (item & 3) * 64 + r0;
                uint32_t r[R];
                const uint64_t g2 = both(gs), e2 = both(ev);
                // The item's first block sets the references; later ones weigh by them as they are, unless a score has outgrown its row's or is the first that its row sees: then
                // the block is gone over a second time, rows without a reference against zero.
                bool set = j < (SPLIT ? 1 : 2);
                while (true) {
                    columns<R>(ts, r);
                    if constexpr (Q8) {                  // both parts of the queries
                        uint32_t second[R];
                        columns<R>(ts + N, second);
#pragma unroll
                        for (int i = 0; i < R; i += 2) {
                            float a, b;
                            apart(add2(pair(r[i], r[i + 1]), pair(second[i], second[i + 1])), a, b);
                            r[i] = __float_as_uint(a);
                            r[i + 1] = __float_as_uint(b);
                        }
                    }
                    if (bad || pos >= total) {
#pragma unroll
                        for (int i = 0; i < R; ++i) r[i] = 0xff800000u;      // -infinity
                    } else if (pos >= len) {
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            if (!((seen[i] >> (pos - len)) & 1)) r[i] = 0xff800000u;
                    }
                    // r = score - reference, in powers of two
                    float m2[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < R; i += 4) {
                        const float4 m = *reinterpret_cast<const float4*>(nr + i);
                        uint64_t a = pair(__float_as_uint(m.x), __float_as_uint(m.y)), b = pair(__float_as_uint(m.z), __float_as_uint(m.w));
                        if constexpr (Q8) { a = add2(a, e2); b = add2(b, e2); }
                        uint64_t s0 = pair(r[i], r[i + 1]), s1 = pair(r[i + 2], r[i + 3]), f0 = g2, f1 = g2;
                        if constexpr (Q8) {
                            const float4 f = *reinterpret_cast<const float4*>(fac + i);
                            s0 = mul2(s0, g2);           // the token's scale first: a row's may be as large as bf16 goes, and only with it is the product the score's size
                            s1 = mul2(s1, g2);
                            f0 = pair(__float_as_uint(f.x), __float_as_uint(f.y));
                            f1 = pair(__float_as_uint(f.z), __float_as_uint(f.w));
                        }
                        float x[4];
                        apart(fma2(s0, f0, a), x[0], x[1]);
                        apart(fma2(s1, f1, b), x[2], x[3]);
                        m2[0] = max3(m2[0], x[0], x[1]);
                        m2[1] = max3(m2[1], x[2], x[3]);
#pragma unroll
                        for (int k = 0; k < 4; ++k) r[i + k] = __float_as_uint(x[k]);
                    }
                    if (set || !group_any(g, fmaxf(m2[0], m2[1]) > GROW + UP)) break;
                    if (tid < R && !known) nr[tid] = 0.f;
                    group_sync(g);
                    set = true;
                }
                if (set) {
                    float v[R];
#pragma unroll
                    for (int i = 0; i < R; ++i) v[i] = __uint_as_float(r[i]);
                    join_lanes<R>(v, lane, [](float a, float b) { return fmaxf(a, b); });
                    if (lane < R) ws[wg * 64 + lane] = v[0];
                    group_sync(g);
                    if (tid < R) {
                        const float mx = fmaxf(fmaxf(ws[tid], ws[64 + tid]), fmaxf(ws[128 + tid], ws[192 + tid]));
                        float down = 0.f, a = 1.f;
                        if (mx > (known ? GROW + UP : -INFINITY)) {
                            down = UP - mx;
                            if (mx + down > UP) down = -mx;          // from 2^27 on UP may be rounded up, at an ulp of 16 beyond what fp16 holds
                            a = known ? exp2f(down) : 0.f;
                            nr[tid] += down;
                            known = true;
                        } else if (!known) {
                            nr[tid] = UNSET;
                        }
                        al[tid] = a;
                        ws[tid] = down;
                    }
                    group_sync(g);
                    // these scores are there, so the product of two blocks ago is done
                    if (SPLIT && j > 0) {
                        ok = wait(&v_empty[(n - 1) % NV], (n - 1) / NV);
                        tc_fence_after();
                    }
                    if (j > (SPLIT ? 0 : 1)) {
                        if (D == 128 || wg < 2) {
#pragma unroll 1
                            for (int x = 0; x < S::P_PARTS; ++x) {
                                uint32_t o[R];
                                columns<R>(to + x * N, o);
#pragma unroll
                                for (int i = 0; i < R; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * al[i]);
#pragma unroll
                                for (int c = 0; c < R / 16; ++c) tmem_st16(to + x * N + 16 * c, o + 16 * c);
                            }
                            tmem_st_wait();
                        }
#pragma unroll
                        for (int i = 0; i < R / 2; ++i) {
                            float a, b;
                            apart(l2[i], a, b);
                            l2[i] = pair(__float_as_uint(a * al[2 * i]), __float_as_uint(b * al[2 * i + 1]));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < R; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) + ws[i]);
                    group_sync(g);                       // `ws` has been read
                }
                uint8_t* pt = sp + buf * S::P_TILE + tid * 128;
                const uint64_t un2 = both(un);
                constexpr int LINE = Q8 ? 16 : 8;        // rows of a 16-byte piece
#pragma unroll
                for (int c = 0; c < R / LINE; ++c) {
                    uint32_t w[LINE / 2], rest[LINE / 2];
#pragma unroll
                    for (int k = 0; k < LINE / 2; ++k) {
                        const int i = LINE * c + 2 * k;
                        const float x = exp2f(__uint_as_float(r[i])), y = exp2f(__uint_as_float(r[i + 1]));
                        const uint64_t xy = pair(__float_as_uint(x), __float_as_uint(y));
                        if constexpr (Q8) l2[i / 2] = fma2(xy, un2, l2[i / 2]);
                        else l2[i / 2] = add2(l2[i / 2], xy);
                        w[k] = pack2<Q8>(x, y);
                        if constexpr (!Q8) rest[k] = pack2_rest(x, y, w[k]);
                    }
                    if constexpr (Q8) {
#pragma unroll
                        for (int x = 0; x < 3; ++x) {
                            const int at = (x * N + r0) / 16 + c;            // piece of the token's line, or two
                            uint32_t t[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) t[k] = top_bytes(w[k]);
                            *reinterpret_cast<uint4*>(pt + (at >> 3) * (BLOCK * 128) + (((at & 7) ^ (tid & 7)) * 16)) =
                                make_uint4(__byte_perm(t[0], t[1], 0x7531), __byte_perm(t[2], t[3], 0x7531), __byte_perm(t[4], t[5], 0x7531), __byte_perm(t[6], t[7], 0x7531));
                            if (x < 2)
#pragma unroll
                                for (int k = 0; k < 8; ++k) w[k] = less_top_bytes(w[k], t[k]);
                        }
                    } else {
                        const int at = c + r0 / 8;               // what is left lies N rows on: in the other half of the line, or in the next line
                        *reinterpret_cast<uint4*>(pt + ((at ^ (tid & 7)) * 16)) = make_uint4(w[0], w[1], w[2], w[3]);
                        *reinterpret_cast<uint4*>(pt + (N == 64 ? BLOCK * 128 : 0) + (((N == 64 ? at : at + N / 8) ^ (tid & 7)) * 16)) = make_uint4(rest[0], rest[1], rest[2], rest[3]);
                    }
                }
                fence_proxy_async();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[buf]);
            }
            // ---- the item's part of this group; the next item's scores are computed meanwhile.  Of an item that no other CTA has a part of the groups join what they
            // have, each for half of the rows
            const Item next = u + it.n < u1 ? item_at(P, starts, u + it.n, u1) : it;
            const bool whole = it.n == it.r.units, shared = !SPLIT && whole && it.n > 1;
            float* wk = P.work + partial_at(P, blockIdx.x, u == u0 ? 0 : 1, SPLIT ? 0 : g, D);
            const float* theirs = wk + (g ? -1 : 1) * (long long)partial_floats(N, D);
            const int rows = max(0, min(N, it.r.nodes * P.G - tile_row(it)) - r0);        // of this group's R
            wk += (size_t)r0 * D;
            float2* ml = reinterpret_cast<float2*>(wk - (size_t)r0 * D + (size_t)N * D) + r0;
            {
                float v[R];
#pragma unroll
                for (int i = 0; i < R / 2; ++i) apart(l2[i], v[2 * i], v[2 * i + 1]);
                join_lanes<R>(v, lane, [](float a, float b) { return a + b; });
                group_sync(g);                           // the maxima have been read
                if (lane < R) ws[wg * 64 + lane] = v[0];
            }
            group_sync(g);
            float2 mine = make_float2(-INFINITY, 0.f);
            if (tid < min(R, rows)) {
                const float sum = (ws[tid] + ws[64 + tid]) + (ws[128 + tid] + ws[192 + tid]);
                if (known) mine = make_float2(UP - nr[tid], sum);
                else if (sum != 0.f) mine = make_float2(0.f, sum);           // scores that are no numbers
            }
            if (tid < min(R, rows)) ml[tid] = mine;
            if (some) ok = wait(&o_full[SPLIT ? 0 : g], o_turn++);
            tc_fence_after();
            uint32_t o[R];
            if (some && (D == 128 || wg < 2)) {
                columns<R>(to, o);
#pragma unroll 1
                for (int x = 1; x < S::P_PARTS; ++x) {
                    uint32_t part[R];
                    columns<R>(to + x * N, part);
#pragma unroll
                    for (int i = 0; i < R; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(part[i]));
                }
                for (unsigned long long left = taint[item & 7]; left; left &= left - 1) {        // values that were cleared: for the rows that see their token
                    const int d = __ffsll((long long)left) - 1, t = len + d;
                    if (t / BLOCK < it.first || t / BLOCK >= it.first + it.n || (!SPLIT && ((t / BLOCK - it.first) & 1) != g)) continue;
                    const int page = P.page_table[(size_t)it.b * P.pt_stride + t / PAGE];
                    if (page < 0 || page >= P.n_pages) continue;
                    const size_t v_at = (((size_t)page * P.Hk + it.kvh) * PAGE + t % PAGE) * D + tid;
                    const uint32_t w = Q8 ? 0x7fffffffu : (uint32_t)reinterpret_cast<const uint16_t*>(P.v_raw)[v_at] << 16;
                    if (Q8 ? (P.v_raw[v_at] & 0x7f) == 0x7f : (w & 0x7f800000u) == 0x7f800000u) {
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            if ((seen_s[(item & 3) * 64 + r0 + i] >> d) & 1) o[i] = __float_as_uint(__uint_as_float(o[i]) + __uint_as_float(w));
                    }
                }
#pragma unroll
                for (int i = 0; i < R; ++i)
                    if (i < rows && (!whole || (shared && (i < R / 2) == (g == 1)))) wk[(size_t)i * D + tid] = __uint_as_float(o[i]);
            }
            if (whole) {
                if (shared) both_sync();
                if (tid < R) {
                    const float2 other = shared && tid < rows ? reinterpret_cast<const float2*>(theirs + (size_t)N * D)[tid] : make_float2(-INFINITY, 0.f);
                    const float top = fmaxf(mine.x, other.x), a = mine.x == -INFINITY ? 0.f : exp2f(mine.x - top), b = other.x == -INFINITY ? 0.f : exp2f(other.x - top);
                    const float sum = mine.y * a + other.y * b, inv = sum != 0.f ? 1.f / sum : 0.f;
                    al[tid] = a * inv;
                    ws[tid] = b * inv;
                }
                group_sync(g);
                if (some && (D == 128 || wg < 2)) {
                    const int at = tile_row(it) + r0;
                    int node = at / P.G, head = at - node * P.G;
                    __nv_bfloat16* out = P.out + (((size_t)it.b * P.T + node) * P.H + it.kvh * P.G) * D + tid;           // head 0 of the node
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        if (i < ((rows + 15) & ~15) && node < P.T && (!shared || (i < R / 2) == (g == 0))) {             // sixteen rows at a time, the ones behind the last are zeros
                            const float a = al[i], b = shared ? ws[i] : 0.f;
                            float y = 0.f;
                            if (a != 0.f) y = __uint_as_float(o[i]) * a;
                            if (b != 0.f) y += theirs[(size_t)i * D + tid] * b;
                            out[(size_t)head * D] = __float2bfloat16_rn(i < rows ? y : 0.f);
                        }
                        if (++head == P.G) { head = 0; ++node; out += (size_t)P.H * D; }
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
        // ------------------------------------------------------------------------------------ queries, values
        regs_dec<REGS_OTHER>();
        const int tid = threadIdx.x - CONVERT_WARP * 32;
        constexpr int EACH = N * D / 8 / 128;            // 16-byte pieces of queries a thread
        uint4 raw[EACH];
        unsigned long long seen = 0, there = 0;
        const uint32_t per_head = 65536 / P.G + 1;
        auto fetch = [&](const Item& it) {
            const int rows = it.r.nodes * P.G - tile_row(it), node0 = tile_row(it) / P.G, head0 = tile_row(it) - node0 * P.G;
            auto node_of = [&](int r) {                  // (head0 + r) / G: below 128 a product and a shift where G is below 64, else 0 or 1
                return node0 + (P.G < 64 ? (int)((head0 + r) * per_head >> 16) : head0 + r >= P.G ? 1 : 0);
            };
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int x = i * 128 + tid, r = x / (D / 8), c = x % (D / 8), node = node_of(r), head = tile_row(it) + r - node * P.G;
                raw[i] = make_uint4(0, 0, 0, 0);
                if (r < rows) raw[i] = *reinterpret_cast<const uint4*>(P.q + (size_t)it.b * P.q_batch + (size_t)node * P.q_row + (size_t)(it.kvh * P.G + head) * D + c * 8);
            }
            seen = there = 0;
            if (tid < min(N, rows)) {                    // joined later: nothing waits for a load here
                const int node = node_of(tid);
                seen = P.mask ? P.mask[(size_t)it.b * P.T + node] : (2ull << node) - 1;
                there = it.r.nodes < 64 ? (1ull << it.r.nodes) - 1 : ~0ull;
            }
        };
        auto put = [&](int item) {
            if (item > 0) ok = wait(q_free, item - 1);   // the products of the last item have read theirs
            if (tid < 64) seen_s[(item & 3) * 64 + tid] = seen & there;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int x = i * 128 + tid, r = x / (D / 8), c = x % (D / 8);
                if constexpr (Q8) {
                    uint32_t w1[2], w2[2], a = 0;
                    const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) a = max(a, max(w[k] & 0x7fffu, (w[k] >> 16) & 0x7fffu));
#pragma unroll
                    for (int o = 1; o < D / 8; o <<= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));      // of the row, which D / 8 neighbouring lanes hold
                    const int e = min(253, max(40, (int)(a >> 7)));          // its biased exponent
                    const float up = pow2(127 + 7 - e);
                    if (c == 0) factor[(item & 3) * 64 + r] = a >= 0x7f80u ? __uint_as_float(0x7fffffffu) : fmaxf(P.scale_log2 * pow2(e - 7 - 127), 1e-30f);       // above zero: it meets -infinity
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
                    *reinterpret_cast<uint2*>(sq + at) = make_uint2(w1[0], w1[1]);
                    *reinterpret_cast<uint2*>(sq + N * D + at) = make_uint2(w2[0], w2[1]);
                } else {
                    *reinterpret_cast<uint4*>(sq + (c / 8) * (N * 128) + r * 128 + (((c & 7) ^ (r & 7)) * 16)) = raw[i];
                }
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
        };
        int n = 0, item = 0;
        Item it{};
        if (u0 < u1) {
            it = item_at(P, starts, u0, u1);
            fetch(it);
            asm volatile("bar.arrive 5, 160;" ::: "memory");
            put(0);
        }
        for (int u = u0; u < u1; ++item) {               // after a wait that ran out as well: the four warps meet at every item
            const int len = it.r.len, total = len + it.r.nodes;
            const bool more = u + it.n < u1;
            const Item next = more ? item_at(P, starts, u + it.n, u1) : it;
            if (more) fetch(next);
            if (tid == 0) taint[item & 7] = 0;           // eight items back: nobody reads it any more
            convert_sync();
            for (int j = 0; j < it.n; ++j, ++n) {
                const int t0 = (it.first + j) * BLOCK, sV = n % NV, t = t0 + tid;
                ok = wait(&v_full[sV], n / NV);
                const bool none = t >= total || (ok && (bad_pages[n & 7] >> (tid >> 6)) & 1);
                if (ok && (t >= len || none)) {          // a drafted token, or none
                    uint8_t* v = sv + sV * S::TILE + (tid >> 6) * (S::TILE / 2) + (tid & 63) * (Q8 ? D : 128);
                    bool odd = false;
                    for (int i = 0; i < S::KEY / 16; ++i) {                  // in any order
                        uint4* w = reinterpret_cast<uint4*>(v + (Q8 ? i * 16 : (i / 8) * 8192 + (i & 7) * 16));
                        if (none) { *w = make_uint4(0, 0, 0, 0); continue; }
                        uint4 x = *w;
                        uint32_t* y = reinterpret_cast<uint32_t*>(&x);
                        uint32_t any = 0;
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t no = Q8 ? __vcmpeq4(y[k] & 0x7f7f7f7fu, 0x7f7f7f7fu) : __vcmpeq2(y[k] & 0x7f807f80u, 0x7f807f80u);
                            any |= no;
                            y[k] &= ~no;
                        }
                        if (any) { *w = x; odd = true; }
                    }
                    if (odd) atomicOr(&taint[item & 7], 1ull << (t - len));
                }
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(&v_ready[sV]);
                ok = __all_sync(0xffffffffu, ok);
            }
            u += it.n;
            if (more) put(item + 1);
            it = next;
        }
        if (!ok) *abort_flag = 1;
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) tmem_dealloc(tmem, S::TMEM);
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

// Partial results of cut items: two a CTA (up to 32 rows) or one; tile_rows is 16, 32 or 64.
template <int D, bool Q8>
int launch_few(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    CUtensorMap mk, mv;
    const long long rows = (long long)p.n_pages * p.Hk * PAGE;
    auto map = [&](CUtensorMap* m, const void* pages) {  // rows of a token; a row of 128 bytes is 64 elements of the map's
        return Q8 && D == 64 ? ptb_make_tmap_64b(m, pages, rows, PAGE) : ptb_make_tmap_bf16(m, pages, Q8 ? 64 : D, rows, Q8 ? 64 : D, 64, PAGE);
    };
    if (map(&mk, k_pages) || map(&mv, v_pages)) return -1;
    if constexpr (Q8)                                    // bf16 pages: mma.sync
        if (p.tile_rows == 16) return launch_n<D, Q8, 16>(p, mk, mv, st);
    return p.tile_rows == 32 ? launch_n<D, Q8, 32>(p, mk, mv, st) : launch_n<D, Q8, 64>(p, mk, mv, st);
}
template int launch_few<64, false>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<64, true>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<128, false>(const Params&, const void*, const void*, cudaStream_t);
template int launch_few<128, true>(const Params&, const void*, const void*, cudaStream_t);

}  // namespace tree
}  // namespace ptb
