// The cache entries of several tokens at once: rotary + page write with the slot apart from the position, in bf16 or quantised on the way, and the
// entries of accepted drafted tokens moved into place.
//
// Quantised pages hold e4m3 values [page][kv_head][64][D] and one biased exponent byte [page][kv_head][64] for each token's keys and values of a head:
//   x = value * 2^(byte - 127),  value = rn_e4m3(x 2^-e),  e = the least integer with max |x| <= 448 2^e, kept in [-64, 64].
// A power of two makes the scaling exact both ways (the one rounding is the one to e4m3, at most 2^-4 of a value) and costs e4m3, which has exponents of
// its own, nothing but the last binade.  Infinities are stored as NaN: neither becomes a value that looks sound.
// A slot outside the table, or a page id outside the pool, is never written: PTB_ERR_BOUNDS goes to the status word.
#include "common.cuh"
#include "ptb200_types.h"
#include <cuda_fp8.h>

namespace ptb {
namespace {

constexpr int PW_PAGE = 64;
constexpr int PW_THREADS = 256;

struct WriteParams {
    const __nv_bfloat16* qkv;      // [n, ld]: q heads, then k heads, then v heads
    long long ld;
    const int* pos;                // [n] position (angle)
    const int* slot;               // [n] place in the sequence's pages; null: the position.  Negative: nothing is stored, and a position outside the tables is no error
    const int* req;                // [n] row of the page table
    const int* page_table;
    int pt_stride, pt_rows, n_pages;
    const float* cos;              // [max_pos, D / 2]
    const float* sin;
    int max_pos;
    __nv_bfloat16* q_out;          // [n, H D]
    __nv_bfloat16* k_out;          // optional [n, Hk, D]
    void* k_pages;
    void* v_pages;
    uint8_t* k_exp;                // [n_pages, Hk, 64], null: bf16 pages
    uint8_t* v_exp;
    int n, H, Hk;
    int* status;
};

__device__ __forceinline__ void unpack8(const uint4& raw, float* f) {
    const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
    for (int i = 0; i < 4; ++i) { const float2 v = __bfloat1622float2(h2[i]); f[2 * i] = v.x; f[2 * i + 1] = v.y; }
}
__device__ __forceinline__ uint4 pack8(const float* f) {
    uint4 o;
    __nv_bfloat162* h2 = reinterpret_cast<__nv_bfloat162*>(&o);
#pragma unroll
    for (int i = 0; i < 4; ++i) h2[i] = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    return o;
}

// Largest magnitude of a token's head over the L neighbouring lanes that hold it, as bits (magnitudes order as integers do; NaN and infinity lie above).
template <int L>
__device__ __forceinline__ uint32_t head_max(const float* f) {
    uint32_t a = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) a = max(a, __float_as_uint(f[i]) & 0x7fffffffu);
#pragma unroll
    for (int o = L / 2; o > 0; o >>= 1) a = max(a, __shfl_xor_sync(0xffffffffu, a, o));
    return a;
}

// The head's exponent, and its sixteen values of this lane in e4m3 (two words each of the low and the high eight).
template <int L>
__device__ __forceinline__ int quantise(float* f, uint2& lo, uint2& hi) {
    uint32_t a = head_max<L>(f);
    if (a >= 0x7f800000u) {                              // infinities become NaN, and neither counts for the exponent.  All lanes of the head agree on a
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if ((__float_as_uint(f[i]) & 0x7fffffffu) >= 0x7f800000u) f[i] = __uint_as_float(0x7fffffffu);
    }
    if (__any_sync(0xffffffffu, a >= 0x7f800000u)) {     // the shuffles need the whole warp
        float g[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = (__float_as_uint(f[i]) & 0x7fffffffu) >= 0x7f800000u ? 0.f : f[i];
        a = head_max<L>(g);
    }
    // a = m 2^k with m in [1, 2): 448 = 1.75 * 2^8
    const int e = min(64, max(-64, (int)(a >> 23) - 127 - 8 + ((a & 0x7fffffu) > 0x600000u ? 1 : 0)));
    const float s = __uint_as_float((uint32_t)(127 - e) << 23);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t p0 = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i] * s, f[4 * i + 1] * s), __NV_SATFINITE, __NV_E4M3);
        const uint32_t p1 = __nv_cvt_float2_to_fp8x2(make_float2(f[4 * i + 2] * s, f[4 * i + 3] * s), __NV_SATFINITE, __NV_E4M3);
        w[i] = p0 | (p1 << 16);
    }
    lo = make_uint2(w[0], w[1]);
    hi = make_uint2(w[2], w[3]);
    return e + 127;
}

// D / 16 lanes a head, eight pairs (or sixteen values of v) a lane, one CTA a token.  Products and sums of the rotation are rounded one by one, so that
// the result does not depend on how the compiler contracts them.  Bound by bytes.
template <int D, bool Q8>
__global__ void __launch_bounds__(PW_THREADS) paged_write_kernel(const __grid_constant__ WriteParams P) {
    constexpr int L = D / 16, PER = PW_THREADS / L, HALF = D / 2;
    pdl_wait();
    pdl_launch_dependents();
    const int i = blockIdx.x, j = threadIdx.x % L, g = threadIdx.x / L;
    const int pos = P.pos[i], slot = P.slot ? P.slot[i] : pos, req = P.req[i];
    const bool angle = pos >= 0 && pos < P.max_pos;
    int page = -1;
    if (slot >= 0 && slot / PW_PAGE < P.pt_stride && req >= 0 && req < P.pt_rows) page = P.page_table[(size_t)req * P.pt_stride + slot / PW_PAGE];
    const bool stored = page >= 0 && page < P.n_pages && angle;
    if (threadIdx.x == 0 && P.status && slot >= 0 && !stored) atomicExch(P.status, PTB_ERR_BOUNDS);
    float c[8], s[8];
    if (angle) {
        const float4 *cs = reinterpret_cast<const float4*>(P.cos + (size_t)pos * HALF) + 2 * j, *sn = reinterpret_cast<const float4*>(P.sin + (size_t)pos * HALF) + 2 * j;
        const float4 c0 = cs[0], c1 = cs[1], s0 = sn[0], s1 = sn[1];
        c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
        s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
    } else {
#pragma unroll
        for (int x = 0; x < 8; ++x) { c[x] = 1.f; s[x] = 0.f; }
    }
    const uint4* row = reinterpret_cast<const uint4*>(P.qkv + (size_t)i * P.ld);
    const int heads = P.H + 2 * P.Hk;
    for (int h0 = 0; h0 < heads; h0 += PER) {            // the whole warp stays in the loop: heads exchange through shuffles
        const int h = h0 + g;
        const bool on = h < heads;
        const int kind = h < P.H ? 0 : h < P.H + P.Hk ? 1 : 2;
        // of v a lane takes the same two pieces, D / 2 apart
        float f[16];
        if (on) {
            const uint4 a = row[h * (D / 8) + j], b = row[h * (D / 8) + L + j];
            unpack8(a, f);
            unpack8(b, f + 8);
        } else {
#pragma unroll
            for (int x = 0; x < 16; ++x) f[x] = 0.f;
        }
        if (kind < 2) {
#pragma unroll
            for (int x = 0; x < 8; ++x) {
                const float a = f[x], b = f[8 + x];
                f[x] = __fsub_rn(__fmul_rn(a, c[x]), __fmul_rn(b, s[x]));
                f[8 + x] = __fadd_rn(__fmul_rn(b, c[x]), __fmul_rn(a, s[x]));
            }
        }
        if (on && kind == 0) {
            uint4* q = reinterpret_cast<uint4*>(P.q_out + ((size_t)i * P.H + h) * D);
            q[j] = pack8(f);
            q[L + j] = pack8(f + 8);
        }
        const int kh = kind == 1 ? h - P.H : h - P.H - P.Hk;
        if (on && kind == 1 && P.k_out) {
            uint4* k = reinterpret_cast<uint4*>(P.k_out + ((size_t)i * P.Hk + kh) * D);
            k[j] = pack8(f);
            k[L + j] = pack8(f + 8);
        }
        const size_t at = ((size_t)(stored ? page : 0) * P.Hk + (kind ? kh : 0)) * PW_PAGE + (stored ? slot % PW_PAGE : 0);
        if constexpr (Q8) {
            uint2 lo, hi;
            const int e = quantise<L>(f, lo, hi);
            if (on && kind && stored) {
                uint2* dst = reinterpret_cast<uint2*>(static_cast<uint8_t*>(kind == 1 ? P.k_pages : P.v_pages) + at * D);
                dst[j] = lo;
                dst[L + j] = hi;
                if (j == 0) (kind == 1 ? P.k_exp : P.v_exp)[at] = (uint8_t)e;
            }
        } else if (on && kind && stored) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(kind == 1 ? P.k_pages : P.v_pages) + at * D);
            dst[j] = pack8(f);
            dst[L + j] = pack8(f + 8);
        }
    }
}

constexpr int KEEP_THREADS = 256, KEEP_AT_ONCE = 4;
constexpr int KEEP_LAYERS = (4096 - 128) / (4 * (int)sizeof(void*));     // as many as the parameters of a launch hold, 4 KB
static_assert(KEEP_THREADS == 64 * KEEP_AT_ONCE, "a thread for each layer and token");

struct KeepParams {
    uint8_t* pool[4][KEEP_LAYERS];       // keys, values, their exponents (or null)
    const int* lens;                     // [B]
    const int* path;                     // [B, T]
    const int* count;                    // [B]
    const int* page_table;
    int pt_stride, n_pages, Hk, row, T, layers;        // row: bytes of a token's keys of a head
    int* status;
};
static_assert(sizeof(KeepParams) <= 4096, "parameters of a launch");

// A block moves the keys (or the values) of one head in up to four layers: threads are (token of the path, 16-byte piece), as many tokens at a time as fit.  A path ascends, so a token never
// moves behind its own place and no later one reads a slot that an earlier one filled; within a group all are read before the first is written.  Latency
// bounds it (a request's path is a few dozen kilobytes a layer), so all layers go in one launch and a move is one chain of four loads.
__global__ void __launch_bounds__(KEEP_THREADS) paged_keep_kernel(const __grid_constant__ KeepParams P) {
    __shared__ int at[2][64];            // where a token comes from and goes to: page * 64 + place, or -1
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, layer0 = blockIdx.z * KEEP_AT_ONCE, which = blockIdx.x & 1, head = blockIdx.x >> 1, tid = threadIdx.x;
    const int n = min(P.count[b], P.T - 1);
    if (n <= 0) return;
    if (tid < 128) {                     // thread (end, token): looks one place up
        const int end = tid >> 6, j = tid & 63;
        int x = -1;
        if (j >= 1 && j <= n) {
            const int from = P.path[(size_t)b * P.T + j];
            if (from < j || from >= P.T) {
                if (P.status) atomicExch(P.status, PTB_ERR_BOUNDS);
            } else if (from != j) {
                const int slot = P.lens[b] + (end ? j : from);
                const int page = slot >= 0 && slot / PW_PAGE < P.pt_stride ? P.page_table[(size_t)b * P.pt_stride + slot / PW_PAGE] : -1;
                if (page >= 0 && page < P.n_pages) x = page * PW_PAGE + slot % PW_PAGE;
                else if (P.status) atomicExch(P.status, PTB_ERR_BOUNDS);
            }
        }
        at[end][j] = x;
    }
    __syncthreads();
    const int per = P.row / 16, together = KEEP_THREADS / per, j0 = tid / per, piece = tid - j0 * per;
    auto spot = [&](int x, int row) { return ((size_t)(x / PW_PAGE) * P.Hk + head) * PW_PAGE * row + (size_t)(x % PW_PAGE) * row; };
    for (int g = 1; g <= n; g += together) {
        const int j = g + j0;
        const bool on = j0 < together && j <= n && at[0][j] >= 0 && at[1][j] >= 0;
        uint4 v[KEEP_AT_ONCE];
#pragma unroll
        for (int l = 0; l < KEEP_AT_ONCE; ++l)
            if (on && layer0 + l < P.layers) v[l] = *reinterpret_cast<const uint4*>(P.pool[which][layer0 + l] + spot(at[0][j], P.row) + piece * 16);
        __syncthreads();
#pragma unroll
        for (int l = 0; l < KEEP_AT_ONCE; ++l)
            if (on && layer0 + l < P.layers) *reinterpret_cast<uint4*>(P.pool[which][layer0 + l] + spot(at[1][j], P.row) + piece * 16) = v[l];
        __syncthreads();
    }
    if (P.pool[2][0]) {                  // thread (layer, token) moves an exponent
        const int l = layer0 + (tid >> 6), j = tid & 63;
        const bool on = l < P.layers && j >= 1 && j <= n && at[0][j] >= 0 && at[1][j] >= 0;
        uint8_t v = 0;
        if (on) v = P.pool[2 + which][l][spot(at[0][j], 1)];
        __syncthreads();
        if (on) P.pool[2 + which][l][spot(at[1][j], 1)] = v;
    }
}

bool off16(const void* p) { return ((uintptr_t)p & 15) != 0; }

}  // namespace
}  // namespace ptb

using namespace ptb;

// Rotate q and k of `n` tokens (pairs (j, j + D/2)); q goes to q_out [n, H D], k and v to the page slots of (req, slot), slot null: the position, negative: not
// stored.  qkv: [n, ld] bf16; cos / sin: [max_pos, D/2] fp32; k_out optional [n, Hk, D]: the rotated keys.  k_exp and v_exp null: bf16 pages
// [n_pages, Hk, 64, D]; else e4m3 pages with one biased exponent byte for a token's keys (values) of a head.  D is 64 or 128.  Tokens of one slot are equal.
PTB_API int ptb_paged_write(const void* qkv, long long ld, int n, int H, int Hk, int D, const int* pos, const int* slot, const int* req, const int* page_table, int pt_stride,
                            int pt_rows, int n_pages, const float* cos, const float* sin, int max_pos, void* q_out, void* k_out, void* k_pages, void* v_pages, void* k_exp,
                            void* v_exp, int* status, cudaStream_t st) {
    if (n <= 0) return 0;
    if ((D != 64 && D != 128) || H < 0 || Hk <= 0) { ptb_set_error("paged_write: head size %d not in {64, 128}, or no heads (%d, %d)", D, H, Hk); return -1; }
    if (ld < (long long)(H + 2 * Hk) * D || ld % 8) { ptb_set_error("paged_write: rows of %lld values for %d heads of %d (a multiple of eight is needed)", ld, H + 2 * Hk, D); return -1; }
    if (off16(qkv) || off16(q_out) || off16(k_out) || off16(k_pages) || off16(v_pages) || off16(cos) || off16(sin)) { ptb_set_error("paged_write: operands need to be 16-byte aligned"); return -1; }
    if (!k_exp != !v_exp) { ptb_set_error("paged_write: exponents of keys and of values belong together"); return -1; }
    WriteParams p;
    p.qkv = (const __nv_bfloat16*)qkv; p.ld = ld; p.pos = pos; p.slot = slot; p.req = req; p.page_table = page_table; p.pt_stride = pt_stride; p.pt_rows = pt_rows;
    p.n_pages = n_pages; p.cos = cos; p.sin = sin; p.max_pos = max_pos; p.q_out = (__nv_bfloat16*)q_out; p.k_out = (__nv_bfloat16*)k_out;
    p.k_pages = k_pages; p.v_pages = v_pages; p.k_exp = (uint8_t*)k_exp; p.v_exp = (uint8_t*)v_exp; p.n = n; p.H = H; p.Hk = Hk; p.status = status;
    void (*k)(WriteParams) = D == 128 ? (k_exp ? paged_write_kernel<128, true> : paged_write_kernel<128, false>) : (k_exp ? paged_write_kernel<64, true> : paged_write_kernel<64, false>);
    PTB_CUDA_OK(ptb_launch(k, dim3(n), dim3(PW_THREADS), 0, st, ptb_pdl_enabled(), p));
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}

// The cache entries of each request's accepted drafted tokens, moved from slot lens[b] + path[b][j] to lens[b] + j for j in 1 .. count[b], in every
// layer.  pools: [4][layers] device pointers (keys, values, their exponents or null), row: bytes of a token's keys of a head; path [B, T] ascends.
PTB_API int ptb_paged_keep(void* const* pools, int layers, int B, int T, int Hk, int row, int n_pages, const int* lens, const int* path, const int* count, const int* page_table,
                           int pt_stride, int* status, cudaStream_t st) {
    if (B <= 0 || layers <= 0 || T <= 1) return 0;
    if (Hk <= 0 || row <= 0 || row % 16 || row > 16 * KEEP_THREADS || B > 65535 || T > 64 || n_pages > 0x7fffffff / PW_PAGE) {
        ptb_set_error("paged_keep: %d kv heads of %d bytes, %d requests of %d nodes (up to 64), %d pages", Hk, row, B, T, n_pages);
        return -1;
    }
    for (int l0 = 0; l0 < layers; l0 += KEEP_LAYERS) {
        const int m = layers - l0 < KEEP_LAYERS ? layers - l0 : KEEP_LAYERS;
        KeepParams p;
        memset(&p, 0, sizeof(p));
        for (int l = 0; l < m; ++l) {
            for (int w = 0; w < 4; ++w) p.pool[w][l] = (uint8_t*)pools[(size_t)w * layers + l0 + l];
            if (!p.pool[0][l] || !p.pool[1][l] || off16(p.pool[0][l]) || off16(p.pool[1][l])) { ptb_set_error("paged_keep: the pools need to be 16-byte aligned"); return -1; }
            if (!p.pool[2][l] != !p.pool[2][0] || !p.pool[3][l] != !p.pool[2][0]) { ptb_set_error("paged_keep: some pools have exponents and some have none"); return -1; }
        }
        p.lens = lens; p.path = path; p.count = count; p.page_table = page_table; p.pt_stride = pt_stride; p.n_pages = n_pages; p.Hk = Hk; p.row = row; p.T = T; p.layers = m; p.status = status;
        PTB_CUDA_OK(ptb_launch(paged_keep_kernel, dim3(2 * Hk, B, (m + KEEP_AT_ONCE - 1) / KEEP_AT_ONCE), dim3(KEEP_THREADS), 0, st, ptb_pdl_enabled(), p));
    }
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}
