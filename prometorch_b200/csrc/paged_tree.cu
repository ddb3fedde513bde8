// Sixteen rows of drafted tokens at a time against a bf16 cache on mma.sync (up to 32 rows in all), the merge of items that were cut, and which kernel takes what; see paged_tree.cuh.
//
// One CTA of eight warps per SM.  A warp takes every eighth piece of sixteen tokens of the CTA's run, keeps an online softmax of its own over them, and joins the others when
// an item ends.  It brings its pieces itself: keys and values of a piece are one TMA box each of 128-byte rows with the 128-byte swizzle, into a ring that only this warp
// reads, so that a stage is free again at a __syncwarp; the rings of an SM hold 128 KB, several times what the memory's latency needs.
//
// S = Q K^T and O = P V are m16n8k16 products whose operands come from shared memory 16 bytes a lane, without a transposing load.  The order of the contraction is
// free as long as both operands keep it, so lane c of a row's four holds whole 16-byte pieces of a key; and output column n of tile t may
// be any head element, so lane r holds one 16-byte piece of a value row for all tiles.  Which of eight tokens lane r takes (`token_of`) is chosen so
// that the eight lanes of a quarter warp fall on the eight 16-byte columns of the swizzled rows, for keys and for values.
//
// A weight is two bf16, itself rounded and what that leaves (at most 2^-16 of it is lost), each a product of its own; scores, maxima, sums and accumulators are fp32.
#include "paged_tree.cuh"

namespace ptb {
namespace tree {
namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32, ROWS = 16, PIECE = 16, PIECES = PAGE / PIECE;

template <int D>
struct Geo {
    static constexpr int ROW = D * 2;                                  // bytes of a token
    static constexpr int BYTES = PIECE * ROW, LINES = BYTES / 128;     // of a piece
    static constexpr int STAGE = 2 * BYTES;                            // keys, values
    static constexpr int STAGES = 16384 / STAGE;                       // 16 KB a warp
    static constexpr int KSTEPS = D / 16, VTILES = D / 8;
    static constexpr int PITCH = D + 8;                                // floats of a row of the joining buffer
    static constexpr int OFF_JOIN = WARPS * STAGES * STAGE;
    static constexpr int OFF_ML = OFF_JOIN + WARPS * ROWS * PITCH * 4, OFF_BAR = OFF_ML + WARPS * ROWS * 8, OFF_PLAN = OFF_BAR + WARPS * STAGES * 8 + 64;
    static constexpr int TOTAL = OFF_PLAN + 1024;                      // and the plan
    static_assert(TOTAL + plan_bytes(MAX_B) <= 227 * 1024, "shared memory of a CTA");
};

// Which of eight neighbouring tokens lane r (0 .. 7) takes; see above.  Keys: lanes 2p and 2p + 1 of one phase differ in the bit that moves a token to the other
// half of a line.  Values: the tokens of lanes 0, 2, 4, 6 (and of 1, 3, 5, 7) fall on four different pairs of columns.
template <int ROW>
__device__ __forceinline__ int token_of(int r) {
    constexpr uint32_t order = ROW == 128 ? 0x37156240u : 0x57463120u;
    return (order >> (4 * r)) & 7;
}
// Offset of byte `at` of token t in a swizzled piece.
template <int ROW>
__device__ __forceinline__ uint32_t place(int t, int at) {
    const uint32_t x = t * ROW + at;
    return x ^ (((x >> 7) & 7) << 4);
}

__device__ __forceinline__ void mma(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void tma_2d(void* dst, const CUtensorMap* map, int c0, int c1, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)),
                 "r"(c0), "r"(c1)
                 : "memory");
}

// Head element of contraction step s, lane c (the first of four), and of output tile t, column n.
__device__ __forceinline__ constexpr int k_elem(int s, int c) { return (s / 4) * 64 + (c + 4 * ((s / 2) & 1)) * 8 + (s & 1) * 4; }
__device__ __forceinline__ constexpr int v_elem(int t, int n) { return (t / 8) * 64 + n * 8 + t % 8; }

// Pieces of an item's part that have tokens.
__device__ __forceinline__ int pieces_of(const Item& it) { return min(it.n * PIECES, (it.r.len + it.r.nodes - it.first * PAGE + PIECE - 1) / PIECE); }

// Piece `count` of a warp's ring.  Where the wait runs out, the pieces behind it that are on their way are waited for as well: nobody leaves while copies arrive in its shared memory.
template <int STAGES>
__device__ __noinline__ bool wait_or_drain(uint64_t* full, int count, int* status) {
    bool ok = mbar_wait(&full[count % STAGES], (uint32_t)((count / STAGES) & 1), status);
    if (!ok)
        for (int k = count; k < count + STAGES; ++k) mbar_wait(&full[k % STAGES], (uint32_t)((k / STAGES) & 1), status);
    return ok;
}

// What a warp still has to fetch: its pieces of the run, one after another, across items.
struct Fetch {
    int u, piece, ids_from, kvh, n, pieces, row, ids;    // ids: this lane's page id, of the warp's pages from ids_from on; row: first entry of the item's pages in the table
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1) paged_tree_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ Params P) {
    using Ge = Geo<D>;
    constexpr int ROW = Ge::ROW;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    float* joined = reinterpret_cast<float*>(smem + Ge::OFF_JOIN);
    float2* ml = reinterpret_cast<float2*>(smem + Ge::OFF_ML);
    int* part = reinterpret_cast<int*>(smem + Ge::OFF_BAR + WARPS * Ge::STAGES * 8);
    int* starts = reinterpret_cast<int*>(smem + Ge::OFF_PLAN);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, c = lane & 3;
    uint8_t* ring = smem + warp * Ge::STAGES * Ge::STAGE;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + Ge::OFF_BAR) + warp * Ge::STAGES;
    if (lane == 0) {
        for (int s = 0; s < Ge::STAGES; ++s) mbar_init(&full[s], 1);
        mbar_fence_init();
    }
    pdl_wait();
    pdl_launch_dependents();
    plan<THREADS>(P, starts, part);
    __syncthreads();
    const int all = starts[P.B], per = units_per_cta(all, P.ctas);
    const int u0 = (int)min((long long)all, (long long)blockIdx.x * per), u1 = min(all, u0 + per);
    if (blockIdx.x == 0)
        for (int b = threadIdx.x; b <= P.B; b += THREADS) P.starts[b] = starts[b];
    if (u0 >= u1) return;

    // ---- fetching: stage s of the ring takes the pieces s, s + STAGES, ... of this warp
    Fetch f;
    uint32_t bad = 0;                                    // stages whose page is none of the pool's
    auto enter = [&](int u) {
        f.u = u;
        if (u < u1) {
            const Item it = item_at(P, starts, u, u1);
            f.kvh = it.kvh; f.n = it.n; f.pieces = pieces_of(it); f.row = it.b * P.pt_stride + it.first; f.piece = warp; f.ids_from = -1;
        }
    };
    auto next = [&] {                                    // to the next piece of this warp
        while (f.u < u1 && f.piece >= f.pieces) enter(f.u + f.n);
    };
    auto fetch = [&](int s) {
        if (f.u >= u1) return;
        const int k = f.piece / WARPS;                   // the item's piece of this warp; its page lies two pages behind the last one's
        if (f.ids_from < 0 || k - f.ids_from >= 32) {
            const int page = (warp + (k + lane) * WARPS) / PIECES;
            f.ids = -1;
            if (page < f.n) {
                f.ids = P.page_table[(size_t)f.row + page];
                if (f.ids < 0 || f.ids >= P.n_pages) {
                    f.ids = -1;
                    if (P.status) atomicExch(P.status, PTB_ERR_BOUNDS);
                }
            }
            f.ids_from = k;
        }
        const int page = __shfl_sync(0xffffffffu, f.ids, k - f.ids_from);
        if (lane == 0) {
            const int head = max(page, 0) * P.Hk + f.kvh, line = head * (PIECES * Ge::LINES) + f.piece % PIECES * Ge::LINES;
            uint8_t* st = ring + s * Ge::STAGE;
            mbar_expect_tx(&full[s], Ge::STAGE);
            tma_2d(st, &tmK, 0, line, &full[s]);
            tma_2d(st + Ge::BYTES, &tmV, 0, line, &full[s]);
        }
        bad = page < 0 ? bad | 1u << s : bad & ~(1u << s);
        f.piece += WARPS;
        next();
    };
    enter(u0);
    next();
#pragma unroll 1
    for (int s = 0; s < Ge::STAGES; ++s) fetch(s);

    // ---- this lane's offsets in a piece: its piece of a key (the first of eight tokens; the second lies eight tokens on), of two values
    constexpr int HALVES = ROW / 64;                     // 64-byte halves of lines of a key row that a row's four lanes cover 16 bytes of each at a time
    uint32_t ko[HALVES], vo[2][ROW / 128];
#pragma unroll
    for (int h = 0; h < HALVES; ++h) ko[h] = place<ROW>(token_of<ROW>(r), h * 64 + c * 16);
#pragma unroll
    for (int h = 0; h < ROW / 128; ++h) {
        vo[0][h] = place<ROW>(token_of<ROW>(2 * c), h * 128 + r * 16);
        vo[1][h] = place<ROW>(token_of<ROW>(2 * c + 1), h * 128 + r * 16);
    }

    int count = 0;
    bool ok = true;
    for (int u = u0; u < u1;) {
        const Item it = item_at(P, starts, u, u1);
        const int len = it.r.len, nodes = it.r.nodes, pieces = pieces_of(it);
        // this lane's two rows
        uint32_t qa[Ge::KSTEPS][4];
        unsigned long long seen[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int row = it.tile * ROWS + r + 8 * x, node = row / P.G, g = row - node * P.G;
            const bool on = node < nodes;
            seen[x] = !on ? 0ull : P.mask ? P.mask[(size_t)it.b * P.T + node] : (2ull << node) - 1;
            const __nv_bfloat16* q = P.q + (size_t)it.b * P.q_batch + (size_t)(on ? node : 0) * P.q_row + (size_t)(it.kvh * P.G + g) * D;
            uint2 raw[Ge::KSTEPS];
#pragma unroll
            for (int s = 0; s < Ge::KSTEPS; ++s) raw[s] = on ? *reinterpret_cast<const uint2*>(q + k_elem(s, c)) : make_uint2(0, 0);
#pragma unroll
            for (int s = 0; s < Ge::KSTEPS; ++s) { qa[s][x] = raw[s].x; qa[s][2 + x] = raw[s].y; }
        }
        float acc[Ge::VTILES][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int t = 0; t < Ge::VTILES; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;

#pragma unroll 1
        for (int piece = warp; piece < pieces; piece += WARPS, ++count) {
            const int s = count % Ge::STAGES, first = it.first * PAGE + piece * PIECE;       // first: the piece's first token
            if (ok && !mbar_try_wait(&full[s], (uint32_t)((count / Ge::STAGES) & 1))) ok = wait_or_drain<Ge::STAGES>(full, count, P.status);
            if (ok && !((bad >> s) & 1)) {
                const uint8_t *sk = ring + s * Ge::STAGE, *sv = sk + Ge::BYTES;
                const bool tail = first + PIECE > len;   // some of its tokens are drafted, or lie behind the last
                float sc[2][4];
                {
                    float part4[2][2][4];                // two chains of products a tile
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 8; ++i) part4[j][i >> 2][i & 3] = 0.f;
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const uint4 w = *reinterpret_cast<const uint4*>(sk + ko[h] + j * 8 * ROW);
                            mma(part4[j][0], qa[2 * h], w.x, w.y);
                            mma(part4[j][1], qa[2 * h + 1], w.z, w.w);
                        }
#pragma unroll
                    for (int j = 0; j < 2; ++j)
#pragma unroll
                        for (int i = 0; i < 4; ++i) sc[j][i] = part4[j][0][i] + part4[j][1][i];
                }
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const int t = 8 * j + token_of<ROW>(2 * c + y);
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float& v = sc[j][2 * x + y];
                            v *= P.scale_log2;
                            if (tail) {
                                const int d = first + t - len;
                                if (d >= 0 && (d >= nodes || !((seen[x] >> d) & 1))) v = -INFINITY;
                            }
                        }
                    }
                // values of this lane's four tokens
                constexpr int VW = ROW / 32;             // words of a lane's piece(s) of a value row
                uint32_t vw[4][VW];
                bool odd = false;                        // a value that is no number, which a row that does not see its token must not meet
#pragma unroll
                for (int k = 0; k < 4; ++k) {
#pragma unroll
                    for (int h = 0; h < VW / 4; ++h) {
                        const uint4 w = *reinterpret_cast<const uint4*>(sv + vo[k & 1][h] + (k >> 1) * 8 * ROW);
                        vw[k][4 * h] = w.x; vw[k][4 * h + 1] = w.y; vw[k][4 * h + 2] = w.z; vw[k][4 * h + 3] = w.w;
                    }
                    if (tail) {
                        const int d = first + 8 * (k >> 1) + token_of<ROW>(2 * c + (k & 1)) - len;
                        if (d >= nodes) {
#pragma unroll
                            for (int i = 0; i < VW; ++i) vw[k][i] = 0;
                        } else if (d >= 0) {
#pragma unroll
                            for (int i = 0; i < VW; ++i) odd |= __vcmpeq2(vw[k][i] & 0x7f807f80u, 0x7f807f80u) != 0;
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
                // a maximum that is passed by less than 2^8 stays the reference: weights grow to 256 at most, and the accumulators are seldom scaled
                if (__any_sync(0xffffffffu, mx[0] > m[0] + 8.f || mx[1] > m[1] + 8.f)) {
                    float g[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const float mn = fmaxf(m[x], mx[x]);
                        g[x] = mn == -INFINITY ? 1.f : exp2f(m[x] - mn);
                        m[x] = mn;
                        l[x] *= g[x];
                    }
#pragma unroll
                    for (int t = 0; t < Ge::VTILES; ++t) { acc[t][0] *= g[0]; acc[t][1] *= g[0]; acc[t][2] *= g[1]; acc[t][3] *= g[1]; }
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
                            l[x] += v;
                        }
                }
                const uint32_t pa[4] = {pack2<false>(sc[0][0], sc[0][1]), pack2<false>(sc[0][2], sc[0][3]), pack2<false>(sc[1][0], sc[1][1]), pack2<false>(sc[1][2], sc[1][3])};
                if (!tail || !__any_sync(0xffffffffu, odd)) {
                    uint32_t rest[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) rest[i] = pack2_rest(sc[i >> 1][2 * (i & 1)], sc[i >> 1][2 * (i & 1) + 1], pa[i]);
#pragma unroll
                    for (int i = 0; i < VW; ++i) {
                        const uint32_t b[4] = {__byte_perm(vw[0][i], vw[1][i], 0x5410), __byte_perm(vw[2][i], vw[3][i], 0x5410), __byte_perm(vw[0][i], vw[1][i], 0x7632),
                                               __byte_perm(vw[2][i], vw[3][i], 0x7632)};
                        mma(acc[2 * i], pa, b[0], b[1]);
                        mma(acc[2 * i + 1], pa, b[2], b[3]);
                        mma(acc[2 * i], rest, b[0], b[1]);
                        mma(acc[2 * i + 1], rest, b[2], b[3]);
                    }
                } else {                                 // token by token, each for the rows that see it
#pragma unroll
                    for (int k = 0; k < 16; ++k) {
                        // token k: accumulator element k % 2 of tile k / 8, of lane r * 4 + k % 8 / 2
                        const int t = (k & 8) + token_of<ROW>(k & 7), from = (lane & ~3) | ((k & 7) >> 1), d = first + t - len;
                        const float w0 = __shfl_sync(0xffffffffu, sc[k >> 3][k & 1], from), w1 = __shfl_sync(0xffffffffu, sc[k >> 3][2 + (k & 1)], from);
                        if (d >= nodes) continue;
                        const bool s0 = d < 0 || ((seen[0] >> d) & 1), s1 = d < 0 || ((seen[1] >> d) & 1);
#pragma unroll
                        for (int tt = 0; tt < Ge::VTILES; ++tt)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int e = v_elem(tt, 2 * c + y);
                                const float v = __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(sv + place<ROW>(t, 2 * e)) << 16);
                                if (s0) acc[tt][y] += w0 * v;
                                if (s1) acc[tt][2 + y] += w1 * v;
                            }
                    }
                }
            }
            __syncwarp();
            if (ok) fetch(s);
        }
        // ---- the item ends here, or the run does: join the warps' parts
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
            const int row = warp * ROWS + r + 8 * x;
            if (c == 0) ml[row] = make_float2(m[x] == -INFINITY && l[x] != 0.f ? 0.f : m[x], l[x]);          // a sum without a maximum is of no numbers
            float* dst = joined + (size_t)row * Ge::PITCH + 2 * c;
#pragma unroll
            for (int t = 0; t < Ge::VTILES; ++t) *reinterpret_cast<float2*>(dst + 8 * t) = make_float2(acc[t][2 * x], acc[t][2 * x + 1]);
        }
        __syncthreads();
        const bool whole = it.n == it.r.units;
        float* wk = P.work + partial_at(P, blockIdx.x, u == u0 ? 0 : 1, 0, D);
        for (int e = threadIdx.x; e < ROWS * D / 2; e += THREADS) {          // two elements a thread
            const int row = e / (D / 2), i = (e - row * (D / 2)) * 2;
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) M = fmaxf(M, ml[k * ROWS + row].x);
            float L = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
            for (int k = 0; k < WARPS; ++k) {
                const float2 q = ml[k * ROWS + row];
                const float g = q.x == -INFINITY ? 0.f : exp2f(q.x - M);
                const float2 a = *reinterpret_cast<const float2*>(joined + (size_t)(k * ROWS + row) * Ge::PITCH + i);
                L += q.x == -INFINITY ? 0.f : q.y * g;
                o0 += q.x == -INFINITY ? 0.f : a.x * g;
                o1 += q.x == -INFINITY ? 0.f : a.y * g;
            }
            // place i of a row: column i % 8 of tile i / 8
            if (whole) {
                const int at = it.tile * ROWS + row, node = at / P.G, g = at - node * P.G;
                if (node < P.T) {
                    const bool on = node < nodes && L != 0.f;
                    __nv_bfloat16* o = P.out + (((size_t)it.b * P.T + node) * P.H + it.kvh * P.G + g) * D;
                    o[v_elem(i / 8, i % 8)] = __float2bfloat16_rn(on ? o0 / L : 0.f);
                    o[v_elem(i / 8, i % 8 + 1)] = __float2bfloat16_rn(on ? o1 / L : 0.f);
                }
            } else {
                *reinterpret_cast<float2*>(wk + ((i / 8) * ROWS + row) * 8 + i % 8) = make_float2(o0, o1);
                if (i == 0) *reinterpret_cast<float2*>(wk + (size_t)ROWS * D + 2 * row) = make_float2(M, L);
            }
        }
        __syncthreads();                                 // the buffer is free again
        u += it.n;
    }
}

// The partial results of items that were cut: one block per sixteen rows of an item, a thread (row, eight columns, every SLICES-th result); and the rows that no unit belongs
// to, which are zeros.  With few blocks a chain of loads is what it costs, and four shorter ones cost less (a chain of 5 behind 540 tokens, both kernels: 14.9 us with one,
// 12.4 with four); with more blocks than the SMs hold, more threads only wait (64 nodes, 8 requests: 9 and 18 us).
// How the accumulators of a partial result lie: TILES [D / 8][rows][8], place i of a row column i % 8 of product tile i / 8;
// EIGHTS the same in the order of the head; ROWWISE [rows][D].
enum Layout { TILES, EIGHTS, ROWWISE };
template <int D, Layout LAYOUT, int SLICES>
__global__ void __launch_bounds__(2 * D * SLICES) paged_tree_merge_kernel(const __grid_constant__ Params P) {
    constexpr int OTHERS = SLICES > 1 ? SLICES - 1 : 1;
    __shared__ float4 share[OTHERS][2][2 * D];
    __shared__ float2 share_ml[OTHERS][2 * D];
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, groups = min(P.tile_rows, (P.T * P.G + 15) / 16 * 16) / 16;
    const int i = blockIdx.x / groups, row0 = (blockIdx.x - i * groups) * 16;
    const int tile = i / P.Hk, kvh = i - tile * P.Hk;
    const Req r = req_of(P, b);
    const int slice = threadIdx.x / (2 * D), tid = threadIdx.x % (2 * D), row = row0 + tid % 16, c8 = tid / 16, at = tile * P.tile_rows + row, node = at / P.G, g = at - node * P.G;
    float o[8], L = 0.f, M = -INFINITY;
#pragma unroll
    for (int x = 0; x < 8; ++x) o[x] = 0.f;
    if (tile < r.tiles && (tile * P.tile_rows + row0) / P.G < r.nodes) {     // some of the sixteen rows are there
        const int per = units_per_cta(P.starts[P.B], P.ctas), a = P.starts[b] + i * r.units, e = a + r.units;
        const int c0 = a / per, c1 = (e - 1) / per, n = (c1 - c0 + 1) * P.parts;
        if (c0 == c1) return;                            // written already
        auto from = [&](int k) {                         // slot 0: the run begins in (or with) this item
            const int c = c0 + k / P.parts;
            return P.work + partial_at(P, c, c * per >= a ? 0 : 1, k % P.parts, D);
        };
        constexpr int AT_ONCE = 4;                       // fetched together, before any of them is needed
        for (int k0 = slice; k0 < n; k0 += AT_ONCE * SLICES) {
            float2 ml[AT_ONCE];
            float4 v[AT_ONCE][2];
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x)
                if (k0 + x * SLICES < n) {
                    const float* p = from(k0 + x * SLICES);
                    ml[x] = *reinterpret_cast<const float2*>(p + (size_t)P.tile_rows * D + 2 * row);
                    const float4* q = reinterpret_cast<const float4*>(p + (LAYOUT == ROWWISE ? (size_t)row * D + c8 * 8 : (size_t)(c8 * P.tile_rows + row) * 8));
                    v[x][0] = q[0];
                    v[x][1] = q[1];
                } else {
                    ml[x] = make_float2(-INFINITY, 0.f);
                }
            float mn = M;
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) mn = fmaxf(mn, ml[x].x);
            const float old = M == -INFINITY ? 0.f : exp2f(M - mn);
            M = mn;
            L *= old;
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] *= old;
#pragma unroll
            for (int x = 0; x < AT_ONCE; ++x) {
                if (ml[x].x == -INFINITY) continue;      // that part saw nothing, and may not have written its accumulators
                const float w = exp2f(ml[x].x - mn);
                L += ml[x].y * w;
                o[0] += v[x][0].x * w; o[1] += v[x][0].y * w; o[2] += v[x][0].z * w; o[3] += v[x][0].w * w;
                o[4] += v[x][1].x * w; o[5] += v[x][1].y * w; o[6] += v[x][1].z * w; o[7] += v[x][1].w * w;
            }
        }
        if constexpr (SLICES > 1) {                      // the slices', in their order
            if (slice > 0) {
                share_ml[slice - 1][tid] = make_float2(M, L);
                share[slice - 1][0][tid] = make_float4(o[0], o[1], o[2], o[3]);
                share[slice - 1][1][tid] = make_float4(o[4], o[5], o[6], o[7]);
            }
            __syncthreads();
            if (slice > 0) return;
            float mn = M;
#pragma unroll
            for (int x = 0; x < SLICES - 1; ++x) mn = fmaxf(mn, share_ml[x][tid].x);
            const float old = M == -INFINITY ? 0.f : exp2f(M - mn);
            L *= old;
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] *= old;
#pragma unroll
            for (int x = 0; x < SLICES - 1; ++x) {
                const float2 ml = share_ml[x][tid];
                if (ml.x == -INFINITY) continue;
                const float w = exp2f(ml.x - mn);
                const float4 a = share[x][0][tid], b = share[x][1][tid];
                L += ml.y * w;
                o[0] += a.x * w; o[1] += a.y * w; o[2] += a.z * w; o[3] += a.w * w;
                o[4] += b.x * w; o[5] += b.y * w; o[6] += b.z * w; o[7] += b.w * w;
            }
        }
    }
    if (slice > 0 || node >= P.T) return;
    const bool on = node < r.nodes && L != 0.f;
    const float inv = on ? 1.f / L : 0.f;
    __nv_bfloat16* out = P.out + (((size_t)b * P.T + node) * P.H + kvh * P.G + g) * D;
    if constexpr (LAYOUT != TILES) {
        uint4 w;
        __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
        for (int x = 0; x < 4; ++x) h[x] = __floats2bfloat162_rn(on ? o[2 * x] * inv : 0.f, on ? o[2 * x + 1] * inv : 0.f);
        *reinterpret_cast<uint4*>(out + 8 * c8) = w;
    } else {
#pragma unroll
        for (int x = 0; x < 8; ++x) out[v_elem(c8, x)] = __float2bfloat16_rn(on ? o[x] * inv : 0.f);
    }
}

template <int D, Layout LAYOUT>
int launch_merge(const Params& p, cudaStream_t st) {
    const int groups = (p.T * p.G + 15) / 16 < p.tile_rows / 16 ? (p.T * p.G + 15) / 16 : p.tile_rows / 16;
    const dim3 grid(p.tiles * p.Hk * groups, p.B);
    if ((int)(grid.x * grid.y) <= p.ctas) PTB_CUDA_OK(ptb_launch(paged_tree_merge_kernel<D, LAYOUT, 4>, grid, dim3(8 * D), 0, st, ptb_pdl_enabled(), p));
    else PTB_CUDA_OK(ptb_launch(paged_tree_merge_kernel<D, LAYOUT, 1>, grid, dim3(2 * D), 0, st, ptb_pdl_enabled(), p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}

template <int D>
int launch_pieces(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    using Ge = Geo<D>;
    CUtensorMap mk, mv;
    const long long lines = (long long)p.n_pages * p.Hk * PIECES * Ge::LINES;
    if (ptb_make_tmap_bf16(&mk, k_pages, 64, lines, 64, 64, Ge::LINES) || ptb_make_tmap_bf16(&mv, v_pages, 64, lines, 64, 64, Ge::LINES)) return -1;
    static bool attr[64];
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        PTB_CUDA_OK(cudaFuncSetAttribute(paged_tree_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Ge::TOTAL + plan_bytes(MAX_B)));
        if (dev < 64) attr[dev] = true;
    }
    PTB_CUDA_OK(ptb_launch(paged_tree_kernel<D>, dim3(p.ctas), dim3(THREADS), (size_t)Ge::TOTAL + plan_bytes(p.B), st, ptb_pdl_enabled(), mk, mv, p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}

int sm_count() {
    static int n = 0;
    if (!n) {
        int dev = 0;
        if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 1;
    }
    return n;
}
// Which kernel, by the rows of a (request, kv head), the type of the pages and how many of those there are: its tile of rows, the tokens of a unit and the partial
// results that a CTA leaves of an item.  Nothing goes by the page table's width, which says how long a request may get and not how long it is.
//   up to 16 rows, bf16: mma.sync.  16 requests of 8192 tokens, 16 rows of 128: 80 us, tokens along the lanes of tensor memory 93; one of 540 tokens, 4 rows: 11.0 and 15.8.
//   up to 32 rows, bf16, and no more items of two tiles each than SMs: mma.sync.  It starts, changes an item and ends in less time, and cuts a long item into smaller pieces; with many
//   items the products in two tiles cost more.  Requests of 60 to 8000 tokens, heads of 64 and 128, 20 or 32 rows: up to 16 items of a kv head it takes 0.72 to 0.87 of the time with the
//   tokens along the lanes on average (one request, 8 kv heads, 20 rows over 540 tokens 12.7 and 16.2 us, over 8000 22 and 32; 2 kv heads, 32 rows over 8000 20 and 50), from 33 to 64 0.91
//   (20 rows) and 0.98 (32; eight requests over 540 tokens 20.0 and 20.9, over 4000 47 and 43), with 256 0.92 and 1.08 (32 requests over 540 tokens, 32 rows: 54 and 49).
//   up to 64 rows: tokens along the lanes.  16 requests of 8192 tokens, bf16, 40 or 64 rows of 128: 92 and 94 us, in tiles of 128 rows 106 and 110; e4m3, 4 rows over 8192 tokens,
//   32 requests: 84, where mma.sync, for which every warp converted what it read, took 148.
//   more, bf16: tiles of 128 rows.
//   more, e4m3: tokens along the lanes, in tiles of 64 rows (see paged_tree_sm100.cu).
struct Choice { int tile_rows, unit, parts; };
Choice choose(int rows, bool q8, long long heads) {
    if (!q8 && (rows <= ROWS || (rows <= 2 * ROWS && 2 * heads <= sm_count()))) return {ROWS, PAGE, 1};
    if (rows > 64) return q8 ? Choice{64, 128, 1} : Choice{128, 128, 2};
    if (rows <= 16) return {16, 128, 2};
    return {rows <= 32 ? 32 : 64, 128, rows <= 32 ? 2 : 1};
}
template <int D, bool Q8>
int launch(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st) {
    if constexpr (!Q8) {
        if (p.tile_rows == 128) return launch_tiles<D>(p, k_pages, v_pages, st) ? -1 : launch_merge<D, EIGHTS>(p, st);
        if (p.unit == PAGE) return launch_pieces<D>(p, k_pages, v_pages, st) ? -1 : launch_merge<D, TILES>(p, st);
    }
    return launch_few<D, Q8>(p, k_pages, v_pages, st) ? -1 : launch_merge<D, ROWWISE>(p, st);
}

}  // namespace
}  // namespace tree
}  // namespace ptb

using namespace ptb;

// Floats of workspace that ptb_paged_attn_tree needs, for either type of pages.
PTB_API long long ptb_paged_tree_work_floats(int B, int T, int H, int Hk, int D) {
    if (Hk <= 0 || T <= 0) return 0;
    long long most = 0;
    for (const bool q8 : {false, true}) {
        const tree::Choice c = tree::choose(T * (H / Hk), q8, (long long)B * Hk);
        const long long n = (long long)tree::sm_count() * 2 * c.parts * (long long)tree::partial_floats(c.tile_rows, D);
        most = n > most ? n : most;
    }
    return most + B + 1;
}

// T drafted tokens of each of B requests (the latest token among them) attend to their request's cached tokens and to one another.  q: [B, T, heads] bf16 with
// pitches in elements, head h at column h * D; out [B, T, H D]; lens [B]: cached tokens before the drafted ones, node i stands in slot lens[b] + i; nodes [B]
// (null: T), rows behind them come out as zeros, as do rows that see nothing; mask [B, T]: bit j, whether the node sees node j (null: a chain).  Pages
// [n_pages, Hk, 64, D]: bf16, or e4m3 with exponents [n_pages, Hk, 64].  D is 64 or 128, T at most 64, B at most 1024.
PTB_API int ptb_paged_attn_tree(const void* q, long long q_batch, long long q_row, void* out, int B, int T, int H, int Hk, int D, const int* lens, const int* nodes, const void* mask,
                                const int* page_table, int pt_stride, int n_pages, const void* k_pages, const void* v_pages, const void* k_exp, const void* v_exp, float scale, float* work,
                                int* status, cudaStream_t st) {
    if (B <= 0) return 0;
    if (T < 1 || T > tree::MAX_NODES || B > tree::MAX_B) { ptb_set_error("paged attention of trees: %d requests of %d nodes (up to %d and %d)", B, T, tree::MAX_B, tree::MAX_NODES); return -1; }
    if (Hk <= 0 || H <= 0 || H % Hk) { ptb_set_error("paged attention of trees: %d heads over %d kv heads", H, Hk); return -1; }
    if (D != 64 && D != 128) { ptb_set_error("paged attention of trees: head size %d not in {64, 128}", D); return -1; }
    if (((uintptr_t)q & 15) || q_batch % 8 || q_row % 8) { ptb_set_error("paged attention of trees: rows of q need to start on 16 bytes"); return -1; }
    if (((uintptr_t)k_pages & 15) || ((uintptr_t)v_pages & 15) || ((uintptr_t)k_exp & 15) || ((uintptr_t)v_exp & 15) || ((uintptr_t)work & 31)) {
        ptb_set_error("paged attention of trees: pools and exponents need to be 16-byte aligned, the workspace 32-byte aligned");
        return -1;
    }
    if (!k_exp != !v_exp) { ptb_set_error("paged attention of trees: exponents of keys and of values belong together"); return -1; }
    if (!(scale > 1e-30f) || !(scale < 1e30f)) { ptb_set_error("paged attention of trees: a scale between 1e-30 and 1e30 is needed"); return -1; }
    if (pt_stride < 1 || n_pages < 1) { ptb_set_error("paged attention of trees: no pages"); return -1; }
    tree::Params p;
    memset(&p, 0, sizeof(p));
    p.q = (const __nv_bfloat16*)q; p.q_batch = q_batch; p.q_row = q_row; p.out = (__nv_bfloat16*)out; p.lens = lens; p.nodes = nodes; p.mask = (const unsigned long long*)mask;
    p.page_table = page_table; p.pt_stride = pt_stride; p.n_pages = n_pages; p.k_exp = (const uint8_t*)k_exp; p.v_exp = (const uint8_t*)v_exp; p.v_raw = (const uint8_t*)v_pages; p.work = work;
    p.B = B; p.T = T; p.H = H; p.Hk = Hk; p.G = H / Hk;
    const tree::Choice c = tree::choose(T * p.G, k_exp != nullptr, (long long)B * Hk);
    p.tile_rows = c.tile_rows;
    p.unit = c.unit;
    p.parts = c.parts;
    p.tiles = (T * p.G + p.tile_rows - 1) / p.tile_rows;
    p.ctas = tree::sm_count();
    p.starts = reinterpret_cast<int*>(work + (size_t)p.ctas * 2 * p.parts * tree::partial_floats(p.tile_rows, D));
    p.scale_log2 = scale * 1.4426950408889634f;
    p.status = status;
    if ((long long)B * p.tiles * Hk * pt_stride > 0x7fffffffll || (long long)n_pages * Hk * 128 > 0x7fffffffll) { ptb_set_error("paged attention of trees: more pages than 31 bits count"); return -1; }
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    PTB_CUDA_OK(cudaSetDevice(dev));     // the tensor-map encoder is a driver call: bind the primary context to this thread
    if (D == 128) return k_exp ? tree::launch<128, true>(p, k_pages, v_pages, st) : tree::launch<128, false>(p, k_pages, v_pages, st);
    return k_exp ? tree::launch<64, true>(p, k_pages, v_pages, st) : tree::launch<64, false>(p, k_pages, v_pages, st);
}
