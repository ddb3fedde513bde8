// What the tcgen05 kernels of paged_tree.cuh share: the cast of warps, tensor memory, pairs of fp32, masks.
#pragma once
#include "paged_tree.cuh"
#include "gemm_sm100.cuh"

namespace ptb {
namespace tree {

using namespace ptb::gemm;

constexpr int BLOCK = 128;                               // tokens of a block: two pages
constexpr int LANES = 128;                               // of tensor memory: rows of a product
// warp 0 brings pages, 1 issues products, 4 .. 11 are two groups of softmax warps, 12 and up prepare tiles
constexpr int SOFTMAX_WARP = 4, CONVERT_WARP = 12;

template <int R> __device__ __forceinline__ void regs_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(R)); }
template <int R> __device__ __forceinline__ void regs_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(R)); }

__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc),
                 "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) { tmem_st16(taddr, r); tmem_st16(taddr + 16, r + 16); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Loads have arrived; the registers are not read before.
__device__ __forceinline__ void tmem_ld_done(uint32_t* r) {
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])::"memory");
}
__device__ __forceinline__ void both_sync() { asm volatile("bar.sync 4, 256;" ::: "memory"); }           // the two softmax groups
__device__ __forceinline__ void convert_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// Pairs of fp32 in one instruction.
__device__ __forceinline__ uint64_t pair(uint32_t x, uint32_t y) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y)); return r; }
__device__ __forceinline__ uint64_t both(float x) { return pair(__float_as_uint(x), __float_as_uint(x)); }
__device__ __forceinline__ void apart(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) { uint64_t r; asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }

// fp16 or bf16 operands, fp32 accumulators.
template <bool FP16>
constexpr uint32_t idesc(int n, int a_mn, int b_mn) { return instr_desc(LANES, n, a_mn, b_mn) & (FP16 ? ~((1u << 7) | (1u << 10)) : ~0u); }

// Which of 32 tokens from `d0` behind the cached ones on (negative: still cached) a row sees; seen: its mask, of nodes that are there.
__device__ __forceinline__ uint32_t visible32(unsigned long long seen, int d0) {
    if (d0 >= 0) return d0 < 64 ? (uint32_t)(seen >> d0) : 0u;
    if (d0 <= -32) return ~0u;
    return ((1u << -d0) - 1) | (uint32_t)(seen << -d0);
}
// A wait ran out, in the block before `blocks`, the loader's last: nobody leaves while copies are on their way into its shared memory.  That block's values were perhaps not sent for (its
// keys neither: their wait is over at once, or runs out as well).
template <int NK, int NV>
__device__ __noinline__ void drain(uint64_t* k_full, uint64_t* v_full, int blocks, int sent_v, int* status) {
    for (int n = max(0, blocks - NK); n < blocks; ++n) mbar_wait(&k_full[n % NK], (uint32_t)((n / NK) & 1), status);
    for (int n = max(0, sent_v - NV); n < sent_v; ++n) mbar_wait(&v_full[n % NV], (uint32_t)((n / NV) & 1), status);
}

// 2^e, for e kept in the range of a normal number.
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(max(-126, min(127, e)) + 127) << 23); }

}  // namespace tree
}  // namespace ptb
