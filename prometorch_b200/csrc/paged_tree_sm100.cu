// More than 64 rows of drafted tokens against a cache in bf16, both products on the 5th-generation tensor cores; see paged_tree.cuh.
//
// One CTA per SM walks its run of units, blocks of 128 tokens (two pages).  Rows lie along the 128 lanes of tensor memory.  Sixteen warps:
//   warp 0      brings keys and values straight to the tiles the products read;
//   warp 1      owns tensor memory and issues S(j) = Q K_j^T and O += P(j) V_j;
//   warps 4-11  softmax, two groups of four warps that take every other block, each with a score buffer, a running maximum and sum and an output accumulator of its
//               own: while one group works on its scores the tensor cores work for the other.  A thread owns a row, so nothing is exchanged.  Weights go back to
//               tensor memory, over the scores they came from, as the first operand of the second product.  The accumulator is scaled, by its own threads, only
//               when a row's maximum has grown by 2^8;
//   warps 12-15 clear the values that must not meet a weight: of drafted tokens, behind the last token, and of pages that are none of the pool's.
//
// What bounds it: the cache's bytes up to 128 rows (a block of 128 keys of 128 elements is 64 KB and takes an SM's share of the memory 1.5 us; exponentials, products and
// softmax instructions take about 0.6 us each, side by side); with more tiles of rows, which fetch the pages again, the products and exponentials.
//
// Weights are rounded to bf16 (by up to 2^-8, without a bias; their sums are of the unrounded ones): the result is off by 2.3e-3 of its norm where rounding the output alone leaves 1.65e-3.
// With what the rounding leaves as a second operand, as the kernels for fewer rows have it, it is 1.65e-3, and 8 trees of 64 over 8191 tokens, 512 rows of 64, take 96 us in place of 66
// (256 rows of 128: 82 and 68), for the softmax's instructions and for the products alike.
//
// e4m3 pages do not come here.  As fp16 tiles, their tokens brought to a common exponent, they were faster with many rows (512 rows of 64 over 8191 tokens: 106 us, with the tokens
// along the lanes 145; 80 over 700: 31 and 27), but one token 2^30 times the others took the others' bits with it, for rows that do not see it as well.
//
// A drafted token that a row does not see must not reach it, whatever it holds: its weight is zero, and zero times a value that is no number is none.  So such values are
// cleared in the tile and the rows that do see the token take them at the end.  What lies behind a request's last token is cleared as well.
#include "paged_tree_sm100.cuh"

namespace ptb {
namespace tree {
namespace {

constexpr int BQ = LANES;
// Registers a thread of the softmax and of the other warps: the launch's shared out anew (512 x 128 = 256 x 184 + 256 x 72).  A softmax thread holds its 128 scores: one wait for tensor
// memory a block in place of eight; 4900 clocks from the scores to the weights became 2000.
constexpr int THREADS = 512, REGS_SOFTMAX = 184, REGS_OTHER = 72;
template <int D>
struct Sm {
    static constexpr int Q_BYTES = BQ * D * 2, TILE = BLOCK * D * 2;
    static constexpr int NK = D == 128 ? 2 : 3, NV = D == 128 ? 3 : 4;
    static constexpr int OFF_K = Q_BYTES, OFF_V = OFF_K + NK * TILE, OFF_BAR = OFF_V + NV * TILE, OFF_PLAN = OFF_BAR + 1024;
    static constexpr int TOTAL = OFF_PLAN + 1024;                      // and the plan
    static_assert(TOTAL + plan_bytes(MAX_B) <= 227 * 1024, "shared memory of a CTA");
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1) paged_tree_tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params P) {
    using S = Sm<D>;
    constexpr int NK = S::NK, NV = S::NV;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t *sq = smem, *sk = smem + S::OFF_K, *sv = smem + S::OFF_V;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::OFF_BAR);
    uint64_t *q_full = bars, *q_free = bars + 1, *s_full = bars + 2, *p_ready = bars + 4, *o_full = bars + 6;            // [1], [1], [2], [2], [2]
    uint64_t *k_full = bars + 8, *k_empty = bars + 12, *v_full = bars + 16, *v_empty = bars + 20, *v_ready = bars + 24;  // [NK], [NK], [NV], [NV], [NV]
    unsigned long long* taint = reinterpret_cast<unsigned long long*>(bars + 28);          // [8] by item: drafted tokens whose values were cleared
    int* bad_pages = reinterpret_cast<int*>(bars + 36);                // [8] by block: bits of pages that are none of the pool's
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
        *abort_flag = 0;
        mbar_fence_init();
        prefetch_tmap(&tmK);
        prefetch_tmap(&tmV);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    constexpr uint32_t TM_S = 0, TM_O = 256;             // two buffers of 128 columns, two of D
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
            // ------------------------------------------------------------------------------------ pages
            int n = 0, sent_v = 0;                           // block of the run; blocks whose values are on their way or there
            for (int u = u0; u < u1 && ok;) {
                const Item it = item_at(P, starts, u, u1);
                const int pages = (it.r.len + it.r.nodes + PAGE - 1) / PAGE;
                for (int j = 0; j < it.n && ok; ++j, ++n) {
                    int id = 0;
                    const int p0 = 2 * (it.first + j);
                    static_assert(PAGE * 2 == BLOCK, "two pages a block");
                    if (lane < 2) {
                        id = p0 + lane < pages ? P.page_table[(size_t)it.b * P.pt_stride + p0 + lane] : 0;
                        if (id < 0 || id >= P.n_pages) {
                            id = -1;
                            if (P.status) atomicExch(P.status, PTB_ERR_BOUNDS);
                        }
                    }
                    const int page[2] = {__shfl_sync(0xffffffffu, id, 0), __shfl_sync(0xffffffffu, id, 1)};
                    if (lane == 0) {
                        const int there = p0 + 1 < pages ? 2 : 1;          // a page that is none of the pool's: any other in its place, which no row sees and whose values are cleared
                        const int sK = n % NK, sV = n % NV;
                        if (n >= NK) ok = wait(&k_empty[sK], n / NK - 1);
                        if (ok) {
                            bad_pages[n & 7] = (page[0] < 0 ? 1 : 0) | (page[1] < 0 ? 2 : 0);
                            mbar_expect_tx(&k_full[sK], there * (S::TILE / 2));
                            for (int x = 0; x < there; ++x)
                                for (int c = 0; c < D / 64; ++c)
                                    tma_load_2d(sk + sK * S::TILE + c * (BLOCK * 128) + x * 8192, &tmK, c * 64, (max(page[x], 0) * P.Hk + it.kvh) * PAGE, &k_full[sK]);
                            if (n >= NV) ok = wait(&v_empty[sV], n / NV - 1);
                        }
                        if (ok) {
                            mbar_expect_tx(&v_full[sV], there * (S::TILE / 2));
                            for (int x = 0; x < there; ++x)
                                for (int c = 0; c < D / 64; ++c)
                                    tma_load_2d(sv + sV * S::TILE + (x * (D / 64) + c) * 8192, &tmV, c * 64, (max(page[x], 0) * P.Hk + it.kvh) * PAGE, &v_full[sV]);
                            sent_v = n + 1;
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
            // ------------------------------------------------------------------------------------ products
            if (lane == 0) {
                constexpr uint32_t id_s = idesc<false>(BLOCK, 0, 0), id_o = idesc<false>(D, 0, 1);
                int base = 0, item = 0, p_turn[2] = {0, 0};  // base: block of the run that the item begins with
                for (int u = u0; u < u1 && ok; ++item) {
                    const Item it = item_at(P, starts, u, u1);
                    const int total = it.r.len + it.r.nodes;
                    auto issue_s = [&](int j) {
                        const int n = base + j, s = n % NK;
                        ok = wait(&k_full[s], n / NK);
                        if (!ok) return;
                        tc_fence_after();
                        const uint64_t a0 = smem_desc(smem_u32(sq), 16, 1024), b0 = smem_desc(smem_u32(sk + s * S::TILE), 16, 1024);          // an address in a descriptor counts 16 bytes
    #pragma unroll
                        for (int c = 0; c < D / 64; ++c)
    #pragma unroll
                            for (int k = 0; k < 4; ++k)
                                umma_bf16(tmem + TM_S + (uint32_t)((j & 1) * BLOCK), a0 + (c * (BQ * 128) + k * 32) / 16, b0 + (c * (BLOCK * 128) + k * 32) / 16, id_s, (c > 0 || k > 0) ? 1u : 0u);
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
                        const uint64_t b0 = smem_desc(smem_u32(sv + s * S::TILE), 8192, 1024);
                        const uint32_t d = tmem + TM_O + (uint32_t)(g * D), p = tmem + TM_S + (uint32_t)(g * BLOCK);
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            if (x == 0 || t0 + PAGE < total)               // the second page is there
#pragma unroll
                                for (int k = 0; k < 4; ++k) umma_ts(d, p + (x * 4 + k) * 8, b0 + (x * (D / 64) * 8192 + k * 2048) / 16, id_o, (j > 1 || x > 0 || k > 0) ? 1u : 0u);
                        umma_commit(&v_empty[s]);
                        if (j + 2 >= it.n) umma_commit(&o_full[g]);
                        if (j + 2 < it.n) issue_s(j + 2);
                    }
                    base += it.n;
                    u += it.n;
                }
                if (!ok) *abort_flag = 1;
            }
        }
    } else if (warp < CONVERT_WARP) {
        // ------------------------------------------------------------------------------------ softmax
        regs_inc<REGS_SOFTMAX>();
        const int g = (warp - SOFTMAX_WARP) >> 2, row = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16), ts = lanes + TM_S + (uint32_t)(g * BLOCK), to = lanes + TM_O + (uint32_t)(g * D);
        int base = 0, s_turn = 0, o_turn = 0;
        const float f = P.scale_log2, grow = 8.f / f;    // weights are powers of two of f times a score less the row's reference m, which lags behind the maximum by no more than `grow`
        // what a thread knows of its row in an item
        struct Row { Item it; bool live, on; unsigned long long seen; };
        auto enter = [&](int u, int item) {
            Row w;
            w.it = item_at(P, starts, u, u1);
            const int rows = min(BQ, w.it.r.nodes * P.G - w.it.tile * BQ), at = w.it.tile * BQ + row;
            w.live = (warp & 3) * 32 < rows;
            w.on = row < rows;
            const int node = w.on ? at / P.G : 0, head = w.on ? at - node * P.G : 0;
            w.seen = 0;
            if (w.on) w.seen = (P.mask ? P.mask[(size_t)w.it.b * P.T + node] : (2ull << node) - 1) & (w.it.r.nodes < 64 ? (1ull << w.it.r.nodes) - 1 : ~0ull);
            if (g == 0) {                                // the first group puts the row of q into the tile
                const uint4* q = reinterpret_cast<const uint4*>(P.q + (size_t)w.it.b * P.q_batch + (size_t)node * P.q_row + (size_t)(w.it.kvh * P.G + head) * D);
                uint4 raw[D / 8];
#pragma unroll
                for (int i = 0; i < D / 8; ++i) raw[i] = w.on ? q[i] : make_uint4(0, 0, 0, 0);
                if (item > 0) ok = wait(q_free, item - 1);                   // the products of the last item have read theirs
#pragma unroll
                for (int i = 0; i < D / 8; ++i) *reinterpret_cast<uint4*>(sq + (i / 8) * (BQ * 128) + row * 128 + (((i & 7) ^ (row & 7)) * 16)) = raw[i];
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            }
            return w;
        };
        Row w;
        if (u0 < u1) w = enter(u0, 0);
        for (int u = u0, item = 0; u < u1; ++item) {
            const Item& it = w.it;
            const int len = it.r.len;
            const bool live = w.live, on = w.on;
            const unsigned long long seen = w.seen;
            float m = -INFINITY, l = 0.f;
            for (int j = g; j < it.n; j += 2) {
                const int n = base + j, t0 = (it.first + j) * BLOCK;
                ok = wait(&s_full[g], s_turn++);
                tc_fence_after();
                if (live && ok) {
                    const int bad = bad_pages[n & 7];
                    const bool some = t0 + BLOCK > len || bad;               // not every row sees every token
                    uint32_t r[BLOCK];                                       // all scores of the block
#pragma unroll
                    for (int c = 0; c < BLOCK / 32; ++c) tmem_ld32(ts + 32 * c, r + 32 * c);
#pragma unroll
                    for (int c = 0; c < BLOCK / 32; ++c) tmem_ld_done(r + 32 * c);
                    if (some) {
#pragma unroll
                        for (int c = 0; c < BLOCK / 32; ++c) {
                            const uint32_t vis = (bad >> (32 * c / PAGE)) & 1 ? 0u : visible32(seen, t0 + 32 * c - len);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!((vis >> i) & 1)) r[32 * c + i] = 0xff800000u;          // -infinity
                        }
                    }
                    float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < BLOCK; i += 2) m4[(i >> 1) & 3] = max3(m4[(i >> 1) & 3], __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
                    const float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    float alpha = 1.f;
                    if (mx > m + grow) {
                        alpha = exp2f((m - mx) * f);
                        m = mx;
                        l *= alpha;
                    }
                    const uint64_t f2 = both(f), mu2 = both(m == -INFINITY ? 0.f : -m);
                    uint64_t l2[2] = {0, 0};
                    // The packed weights take the place of the scores, in registers and in tensor memory.  The reference is taken off before the scale: as one fused product and sum, against a
                    // rounded product, the largest of scores around 2^31 would lie above its own reference by more than fp32 holds
#pragma unroll
                    for (int c = 0; c < BLOCK / 32; ++c) {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            float x, y;
                            apart(mul2(add2(pair(r[32 * c + 2 * i], r[32 * c + 2 * i + 1]), mu2), f2), x, y);
                            x = exp2f(x);
                            y = exp2f(y);
                            l2[i & 1] = add2(l2[i & 1], pair(__float_as_uint(x), __float_as_uint(y)));
                            r[16 * c + i] = pack2<false>(x, y);
                        }
                        tmem_st16(ts + 16 * c, r + 16 * c);
                    }
                    float lx[4];
                    apart(l2[0], lx[0], lx[1]);
                    apart(l2[1], lx[2], lx[3]);
                    l += (lx[0] + lx[1]) + (lx[2] + lx[3]);
                    if (j > 1 && __any_sync(0xffffffffu, alpha != 1.f)) {    // these scores are there, so the product before them is done
#pragma unroll
                        for (int c = 0; c < D / 32; ++c) {
                            tmem_ld32(to + 32 * c, r);
                            tmem_ld_done(r);
#pragma unroll
                            for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
                            tmem_st32(to + 32 * c, r);
                        }
                    }
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_ready[g]);
            }
            // ---- the item's part of this group; the next item's scores are computed meanwhile
            float* wk = P.work + partial_at(P, blockIdx.x, u == u0 ? 0 : 1, g, D);
            float2* ml = reinterpret_cast<float2*>(wk + (size_t)BQ * D) + row;
            Row next = w;
            if (u + it.n < u1) next = enter(u + it.n, item + 1);
            if (it.n > g) ok = wait(&o_full[g], o_turn++);
            tc_fence_after();
            const unsigned long long meets = taint[item & 7] & seen;
            uint32_t r[32];
            auto columns = [&](int c) {                  // 32 of the accumulator's, from 32 c on
                tmem_ld32(to + 32 * c, r);
                tmem_ld_done(r);
                for (unsigned long long left = meets; left; left &= left - 1) {      // values that were cleared, of a token that this row sees
                    const int t = len + __ffsll((long long)left) - 1;
                    if (t / BLOCK < it.first || t / BLOCK >= it.first + it.n || ((t / BLOCK - it.first) & 1) != g) continue;
                    const int page = P.page_table[(size_t)it.b * P.pt_stride + t / PAGE];
                    if (page < 0 || page >= P.n_pages) continue;
                    const size_t v = (((size_t)page * P.Hk + it.kvh) * PAGE + t % PAGE) * D + 32 * c;
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const uint32_t x = (uint32_t)reinterpret_cast<const uint16_t*>(P.v_raw)[v + i] << 16;
                        if ((x & 0x7f800000u) == 0x7f800000u) r[i] = __float_as_uint(__uint_as_float(r[i]) + __uint_as_float(x));
                    }
                }
            };
            // Of an item that no other CTA has a part of, the groups join their parts here, each for half of the columns.
            const bool whole = it.n == it.r.units, shared = whole && it.n > 1;
            if (live && it.n > g && (!whole || shared)) {
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    if (whole && (c < D / 64) == (g == 0)) continue;
                    columns(c);
                    if (on) {
                        float* dst = wk + (4 * c * BQ + row) * 8;
#pragma unroll
                        for (int i = 0; i < 32; i += 8) st_global_32(dst + i * BQ, make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]), make_uint4(r[i + 4], r[i + 5], r[i + 6], r[i + 7]));
                    }
                }
            }
            const float2 mine = on && it.n > g ? make_float2(m == -INFINITY && l != 0.f ? 0.f : m * f, l) : make_float2(-INFINITY, 0.f);      // a sum without a maximum is of no numbers
            if (live) *ml = mine;
            if (shared) both_sync();
            if (whole && live && it.n > g) {
                const float* theirs = wk + (g ? -1 : 1) * (long long)partial_floats(BQ, D);
                const float2 other = shared ? *reinterpret_cast<const float2*>(theirs + (size_t)BQ * D + 2 * row) : make_float2(-INFINITY, 0.f);
                const float top = fmaxf(mine.x, other.x), a = mine.x == -INFINITY ? 0.f : exp2f(mine.x - top), b = other.x == -INFINITY ? 0.f : exp2f(other.x - top);
                const float sum = mine.y * a + other.y * b, inv = sum != 0.f ? 1.f / sum : 0.f;
                const int at = it.tile * BQ + row, node = at / P.G, first = (at & ~15) / P.G;
                const bool put = node < P.T && first < it.r.nodes;           // sixteen rows at a time, the ones behind the last are zeros
                __nv_bfloat16* out = P.out + (((size_t)it.b * P.T + node) * P.H + it.kvh * P.G + (at - node * P.G)) * D;
#pragma unroll 1
                for (int c = 0; c < D / 32; ++c) {
                    if (shared && (c < D / 64) == (g == 1)) continue;
                    columns(c);
                    if (!put) continue;
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        float y[8], z[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                        if (b != 0.f) {
                            const float4* q = reinterpret_cast<const float4*>(theirs + (size_t)((4 * c + i / 8) * BQ + row) * 8);
                            const float4 q0 = q[0], q1 = q[1];
                            z[0] = q0.x; z[1] = q0.y; z[2] = q0.z; z[3] = q0.w; z[4] = q1.x; z[5] = q1.y; z[6] = q1.z; z[7] = q1.w;
                        }
                        uint4 h;
                        __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&h);
#pragma unroll
                        for (int k = 0; k < 8; ++k) y[k] = (a != 0.f ? __uint_as_float(r[i + k]) * (a * inv) : 0.f) + (b != 0.f ? z[k] * (b * inv) : 0.f);
#pragma unroll
                        for (int k = 0; k < 4; ++k) h2[k] = __floats2bfloat162_rn(on ? y[2 * k] : 0.f, on ? y[2 * k + 1] : 0.f);
                        *reinterpret_cast<uint4*>(out + 32 * c + i) = h;
                    }
                }
            }
            tc_fence_before();
            both_sync();                                 // that part has been read; and neither group is more than an item ahead of the other
            base += it.n;
            u += it.n;
            w = next;
        }
        if (!ok) *abort_flag = 1;
    } else {
        // ------------------------------------------------------------------------------------ tiles
        regs_dec<REGS_OTHER>();
        const int tid = (threadIdx.x - CONVERT_WARP * 32) & 127;
        int n = 0, item = 0;
        for (int u = u0; u < u1; ++item) {               // after a wait that ran out as well: the four warps meet at every item
            const Item it = item_at(P, starts, u, u1);
            const int len = it.r.len, total = len + it.r.nodes;
            if (tid == 0) taint[item & 7] = 0;           // eight items back: nobody reads it any more
            convert_sync();
            for (int j = 0; j < it.n; ++j, ++n) {
                const int t0 = (it.first + j) * BLOCK, sV = n % NV, t = t0 + tid;
                ok = wait(&v_full[sV], n / NV);
                const bool none = t >= total || (ok && (bad_pages[n & 7] >> (tid >> 6)) & 1);
                if (ok && (t >= len || none)) {          // a drafted token, or none
                    uint8_t* v = sv + sV * S::TILE + (tid >> 6) * (D / 64) * 8192 + (tid & 63) * 128;
                    bool odd = false;
                    for (int i = 0; i < D / 8; ++i) {
                        uint4* w = reinterpret_cast<uint4*>(v + (i / 8) * 8192 + (i & 7) * 16);
                        if (none) { *w = make_uint4(0, 0, 0, 0); continue; }
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
    if (warp == 1) tmem_dealloc(tmem, 512);
}

}  // namespace

// All items' partial results, two for each CTA and item.
template <int D>
int launch_tiles(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    using S = Sm<D>;
    CUtensorMap mk, mv;
    const long long rows = (long long)p.n_pages * p.Hk * PAGE;
    if (ptb_make_tmap_bf16(&mk, k_pages, D, rows, D, 64, PAGE) || ptb_make_tmap_bf16(&mv, v_pages, D, rows, D, 64, PAGE)) return -1;
    static bool attr[64];
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        PTB_CUDA_OK(cudaFuncSetAttribute(paged_tree_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::TOTAL + plan_bytes(MAX_B)));
        if (dev < 64) attr[dev] = true;
    }
    PTB_CUDA_OK(ptb_launch(paged_tree_tiles_kernel<D>, dim3(p.ctas), dim3(THREADS), (size_t)S::TOTAL + plan_bytes(p.B), st, ptb_pdl_enabled(), mk, mv, p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}
template int launch_tiles<64>(const Params&, const void*, const void*, cudaStream_t);
template int launch_tiles<128>(const Params&, const void*, const void*, cudaStream_t);

}  // namespace tree
}  // namespace ptb
