// Attention of several drafted tokens a request (a tree or a chain; one token: the plain decode step) over a paged cache, bf16 or e4m3.
//
//   o_i = sum_j softmax_j(scale q_i k_j) v_j   over the lens[b] cached tokens and those drafted ones whose bit is set in mask[b][i]
//
// Node i of a request stands in slot lens[b] + i.  All nodes and all query heads of a kv head are rows of one matrix, row = node * G + head, so that
// a page is fetched once for all of them.
//
// Work is dealt on the device: an item is a (request, tile of rows, kv head), a unit 64 or 128 of its tokens; the units of all items, in order, are cut into equal
// runs, one for each CTA.  Lengths differ as they like, the host knows none of them, and a captured graph serves all.  Of an item that is cut every CTA leaves
// a partial result (accumulators, maximum, sum) for paged_tree_merge_kernel.
#pragma once
#include "common.cuh"
#include <cuda.h>

int ptb_make_tmap_bf16(CUtensorMap* map, const void* base, long long inner, long long outer, long long ld, int box_inner, int box_outer);

namespace ptb {
namespace tree {

constexpr int PAGE = 64;
constexpr int MAX_NODES = 64;
constexpr int MAX_B = 1024;

struct Params {
    const __nv_bfloat16* q;              // [B, T, q_row] pitches in elements; head h at column h * D
    long long q_batch, q_row;
    __nv_bfloat16* out;                  // [B, T, H D]
    const int* lens;                     // [B] cached tokens before the drafted ones
    const int* nodes;                    // [B] or null: T
    const unsigned long long* mask;      // [B, T] or null: a chain (node i sees 0 .. i)
    const int* page_table;
    int pt_stride, n_pages;
    const uint8_t* k_exp;                // [n_pages, Hk, 64] biased exponents, null: bf16 pages
    const uint8_t* v_exp;
    const uint8_t* v_raw;                // the pool of values, as bytes
    float* work;                         // partial results of items
    int* starts;                         // [B + 1], behind them: units before each request
    int B, T, H, Hk, G;
    int tile_rows, tiles;                // rows of a tile, tiles of T nodes
    int unit;                            // tokens of a unit
    int parts;                           // partial results that a CTA leaves of an item (of which some may be empty)
    int ctas;
    float scale_log2;
    int* status;
};

__host__ __device__ constexpr size_t partial_floats(int rows, int D) { return (size_t)rows * (D + 2); }

__device__ __forceinline__ int nodes_of(const Params& P, int b) { return P.nodes ? max(0, min(P.nodes[b], P.T)) : P.T; }
__device__ __forceinline__ int cached_of(const Params& P, int b, int n) { return max(0, min(P.lens[b], P.pt_stride * PAGE - n)); }

// What a request asks for: tiles with rows, units of an item.
struct Req { int nodes, len, tiles, units; };
__device__ __forceinline__ Req req_with(const Params& P, int len, int nodes) {
    Req r;
    r.nodes = nodes;
    r.len = len;
    r.tiles = (r.nodes * P.G + P.tile_rows - 1) / P.tile_rows;
    r.units = (r.len + r.nodes + P.unit - 1) / P.unit;
    return r;
}
__device__ __forceinline__ Req req_of(const Params& P, int b) {
    const int nodes = nodes_of(P, b);
    return req_with(P, cached_of(P, b, nodes), nodes);
}
__device__ __forceinline__ int units_of(const Params& P, const Req& r) { return r.tiles * P.Hk * r.units; }

// The plan, in shared memory: starts[b], units before request b (starts[B]: all), and behind them each request's cached tokens and nodes (bytes).
__host__ __device__ constexpr int plan_bytes(int B) { return (2 * B + 1) * 4 + B; }
__device__ __forceinline__ uint8_t* plan_nodes(const Params& P, int* starts) { return reinterpret_cast<uint8_t*>(starts + 2 * P.B + 1); }
// The block's N threads make it, with `part` of N / 32 ints.
template <int N>
__device__ __forceinline__ void plan(const Params& P, int* starts, int* part) {
    int carry = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b0 = 0; b0 < P.B; b0 += N) {
        const int b = b0 + (int)threadIdx.x;
        int u = 0;
        if (b < P.B) {
            const Req r = req_of(P, b);
            u = units_of(P, r);
            starts[P.B + 1 + b] = r.len;
            plan_nodes(P, starts)[b] = (uint8_t)r.nodes;
        }
        int upto = u;
        if (b < P.B && P.status && (P.lens[b] < 0 || P.lens[b] > P.pt_stride * PAGE - nodes_of(P, b))) atomicExch(P.status, PTB_ERR_BOUNDS);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) part[warp] = upto;
        __syncthreads();
        int before = carry, all = carry;
        for (int w = 0; w < N / 32; ++w) {
            if (w == warp) before = all;
            all += part[w];
        }
        if (b < P.B) starts[b + 1] = before + upto;
        if (b == 0) starts[0] = 0;
        carry = all;
        __syncthreads();
    }
}

// The run of units of a CTA: `per` each.
__device__ __forceinline__ int units_per_cta(int all, int ctas) { return max(1, (all + ctas - 1) / ctas); }

// A CTA leaves partial results of at most two items that it shares with others: the one its run begins in (slot 0) and the one it ends in (slot 1; where both are the same,
// slot 0).  An item that it has to itself it writes out.  One result is rows x D accumulators, then [rows] (maximum, sum).
__device__ __forceinline__ size_t partial_at(const Params& P, int cta, int slot, int part, int D) { return (size_t)((cta * 2 + slot) * P.parts + part) * partial_floats(P.tile_rows, D); }

// An item and the part of it in a CTA's run: n units from `first` on.
struct Item { int b, tile, kvh, first, n; Req r; };
__device__ __forceinline__ Item item_at(const Params& P, int* starts, int u, int u1) {
    int lo = 0, hi = P.B;                                // the last request that starts at or before u (empty ones share a start with the next)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= u) lo = mid; else hi = mid;
    }
    Item it;
    it.b = lo;
    it.r = req_with(P, starts[P.B + 1 + lo], plan_nodes(P, starts)[lo]);
    const int in = u - starts[lo], i = in / it.r.units;
    it.first = in - i * it.r.units;
    it.n = min(it.r.units - it.first, u1 - u);
    it.tile = i / P.Hk;
    it.kvh = i - it.tile * P.Hk;
    return it;
}

// Two e4m3 values (the low 16 bits) as fp16, exactly.
__device__ __forceinline__ uint32_t e4m3x2(uint32_t two) {
    uint32_t h;
    asm("{\n .reg .b16 lo;\n cvt.u16.u32 lo, %1;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n}" : "=r"(h) : "r"(two));
    return h;
}
// Two fp32 as e4m3 (the low 16 bits), rounded to nearest.
__device__ __forceinline__ uint32_t e4m3_pack(float x, float y) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(x), "f"(y));
    return r;
}
template <bool Q8>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    uint32_t r;
    if constexpr (Q8) { const __half2 h = __floats2half2_rn(x, y); memcpy(&r, &h, 4); }
    else { const __nv_bfloat162 h = __floats2bfloat162_rn(x, y); memcpy(&r, &h, 4); }
    return r;
}

// What two packed bf16 leave of two fp32, in bf16: sixteen bits of each between them.
__device__ __forceinline__ uint32_t pack2_rest(float x, float y, uint32_t packed) {
    return pack2<false>(x - __uint_as_float(packed << 16), y - __uint_as_float(packed & 0xffff0000u));
}

template <int D> int launch_tiles(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st);               // paged_tree_sm100.cu: bf16
template <int D, bool Q8> int launch_few(const Params& p, const void* k_pages, const void* v_pages, cudaStream_t st);        // paged_tree_few_sm100.cu

}  // namespace tree
}  // namespace ptb
