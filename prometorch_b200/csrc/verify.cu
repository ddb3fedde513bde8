// Which of the drafted tokens a target model keeps, from its logits, the draft's probabilities and given uniform numbers.
//
// Node i of a request holds a drafted token (node 0 the latest token of the sequence) and the target's logits behind it; p_i = softmax(logits_i / temperature).
// The walk starts at node 0.  At node s its children are tried in order:
//   without draft probabilities (tokens proposed outright, several to a parent):  child c is accepted iff u_c (1 - R) < p_s(x_c), R the mass of the children rejected before it;
//   with them (a chain; q_s is what the child was drawn from):                   iff u_c q_s(x_c) < p_s(x_c).
// It goes on at the accepted child.  Where none is left, the last token is drawn with u_0 by the inverse of the cumulative distribution: of p_s without the rejected tokens, or of
// max(p_s - q_s, 0) where a child was rejected; both leave the target's distribution as it is.  Temperature 0 or below (or no number) takes the arg-max (the lowest of equals) throughout.
//
// Two launches.  verify_stats_kernel reads every logit once: a chunk's maximum, its place, and the sum of exponentials, in fp32 (a row's sum is right to about 2^-22; a draft whose number
// lies that near the border of its acceptance may fall on either side).  The bytes of the logits bound it: 41 us for 32 rows of 16 nodes and 151936 tokens, 89 % of the copy rate.
// verify_walk_kernel, a cluster per request, joins the chunks, walks, and draws from one row.  A draw has to fall on the same token for everybody, so that row's weights and
// sums are held in fp64 (an fp32 cumulative sum over 150000 tokens is off by more than a token's share).  Shared memory keeps the logits, half of the weights' size, and
// two CTAs share an SM: a batch of 32 rows of 151936 is one wave (with the weights there, one CTA an SM, it was two: both launches 80 us, now 69).  No unit is full in it (fp64 19 % of
// its cycles, issue 45 %): it is a chain of the chunks' loads, the row's, a pass of exponentials in runs (two against a draft's probabilities) and cluster barriers;
// both launches take 19.5 us for 8 chains of 5 over 32000 tokens.
#include "common.cuh"
#include <math.h>

namespace ptb {
namespace {

constexpr int VF_THREADS = 256, VF_EACH = 32, VF_CHUNK = VF_THREADS * VF_EACH;
constexpr int VF_NODES = 64, VF_ROWS = 65536;      // nodes of a request, and of all: what the attention of trees takes
constexpr int VF_CLUSTER = 16, VF_TOGETHER = 4;
constexpr int VF_WIDE = 128;                 // CTAs of clusters of eight that surely find SMs of their own
constexpr int VF_SLICE = 27 * 1024;          // logits, and the draft's probabilities, that a CTA can hold

struct VerifyParams {
    const void* logits;              // [B, T, V] fp32 or bf16
    long long l_batch, l_row;        // pitches in elements
    const float* probs;              // [B, T, V] or null
    long long p_batch, p_row;
    const int* tokens;               // [B, T]
    const int* parents;              // [B, T] or null: a chain
    const int* nodes;                // [B] or null: T
    const float* u;                  // [B, T]
    const float* temperature;        // [B]
    float4* stats;                   // [B, T, chunks]: maximum, sum, place of the maximum
    int* path;                       // [B, T]
    int* count;                      // [B]
    int* out;                        // [B, T]
    int B, T, V, chunks, slice;      // slice: tokens per CTA of the cluster
};

__device__ __forceinline__ float clean(float l) { return fmaxf(l, -INFINITY); }         // NaN is no token's logit

template <bool BF16>
__device__ __forceinline__ float logit_at(const VerifyParams& P, int b, int i, int v) {
    const size_t at = (size_t)b * P.l_batch + (size_t)i * P.l_row + v;
    return clean(BF16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(P.logits)[at]) : static_cast<const float*>(P.logits)[at]);
}
__device__ __forceinline__ int nodes_of(const VerifyParams& P, int b) { return P.nodes ? max(0, min(P.nodes[b], P.T)) : P.T; }

// Hotter ones count as 2^126, the last whose reciprocal is a normal number in fp32: what a difference of logits is multiplied by stays above zero, and one of -infinity weighs nothing.
__device__ __forceinline__ float temperature_of(const VerifyParams& P, int b) {
    const float t = P.temperature[b];
    return t > 0x1p126f ? 0x1p126f : t;                        // no number stays none
}

// One chunk of one row: maximum, its first place, sum of exp((l - maximum) / temperature).  VEC: rows start on 16 bytes.  Bound by the logits' bytes as long as an element
// costs few instructions: the place is looked for only in the warps that hold the chunk's maximum.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(VF_THREADS) verify_stats_kernel(const __grid_constant__ VerifyParams P) {
    __shared__ float part_m[VF_THREADS / 32], part_s[VF_THREADS / 32];
    __shared__ int place;
    pdl_wait();
    pdl_launch_dependents();
    const int row = blockIdx.x / P.chunks, b = row / P.T, i = row - b * P.T, chunk = blockIdx.x - row * P.chunks, tid = threadIdx.x;
    if (i >= nodes_of(P, b)) return;
    if (tid == 0) place = 0x7fffffff;
    const float t = temperature_of(P, b), scale = (t > 0.f ? __frcp_rn(t) : 1.f) * 1.4426950408889634f;
    const size_t base = (size_t)b * P.l_batch + (size_t)i * P.l_row;
    const int v0 = chunk * VF_CHUNK;
    constexpr int W = !VEC ? 1 : BF16 ? 8 : 4;                 // neighbours that a thread has at once: element k stands at v0 + ((k / W) * VF_THREADS + tid) * W + k % W
    float l[VF_EACH];
#pragma unroll
    for (int g = 0; g < VF_EACH / W; ++g) {
        const int v = v0 + (g * VF_THREADS + tid) * W;
        if (VEC && v + W <= P.V) {
            if constexpr (BF16) {
                const uint4 raw = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(P.logits) + base + v);
                const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
                for (int x = 0; x < W / 2; ++x) { const float2 f = __bfloat1622float2(h2[x]); l[g * W + 2 * x] = f.x; l[g * W + (2 * x + 1) % W] = f.y; }
            } else if constexpr (VEC) {
                const float4 f = *reinterpret_cast<const float4*>(static_cast<const float*>(P.logits) + base + v);
                l[g * W] = f.x; l[g * W + 1 % W] = f.y; l[g * W + 2 % W] = f.z; l[g * W + 3 % W] = f.w;
            }
        } else {
#pragma unroll
            for (int x = 0; x < W; ++x) l[g * W + x] = v + x < P.V ? logit_at<BF16>(P, b, i, v + x) : -INFINITY;
        }
    }
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < VF_EACH; ++k) { l[k] = clean(l[k]); m = fmaxf(m, l[k]); }
    const float mine = m;
    m = warp_max(m);                                           // the reference of the warp's exponentials
    float s = 0.f;
    if (fabsf(m) < INFINITY) {
#pragma unroll
        for (int k = 0; k < VF_EACH; ++k) s += exp2f((l[k] - m) * scale);
    } else if (m > 0.f) {                                      // of infinite logits each counts as one, the others as none
#pragma unroll
        for (int k = 0; k < VF_EACH; ++k) s += l[k] == m ? 1.f : 0.f;
    }
    s = warp_sum(s);
    if ((tid & 31) == 0) { part_m[tid >> 5] = m; part_s[tid >> 5] = s; }
    __syncthreads();
    float top = part_m[0], sum = 0.f;
#pragma unroll
    for (int w = 1; w < VF_THREADS / 32; ++w) top = fmaxf(top, part_m[w]);
    if (mine == top) {
        int at = 0x7fffffff;
#pragma unroll
        for (int k = VF_EACH - 1; k >= 0; --k)
            if (l[k] == top) at = v0 + ((k / W) * VF_THREADS + tid) * W + k % W;
        atomicMin(&place, at);
    }
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 0; w < VF_THREADS / 32; ++w) sum += part_m[w] == top ? part_s[w] : part_s[w] * exp2f((part_m[w] - top) * scale);
        P.stats[(size_t)row * P.chunks + chunk] = make_float4(top, sum, __int_as_float(place), 0.f);
    }
}

__device__ __forceinline__ double weight(float l, float m, double inv) { return l == -INFINITY ? 0.0 : l == m ? 1.0 : exp(((double)l - (double)m) * inv); }
__device__ __forceinline__ void cluster_sync() { asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ double ld_cluster_f64(uint32_t addr, uint32_t rank) {
    double v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f64 %0, [a];\n}" : "=d"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}
// Sum over the block, the same for every thread (and in every order of arrival).
template <int W>
__device__ __forceinline__ double block_sum(double v, double* part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int i = 0; i < W / 32; ++i) v += part[i];
    return v;
}

// One cluster a request; each CTA of it walks by itself (the tree is small) and holds `slice` logits of the row that the last token is drawn from.
template <bool BF16, int W>
__global__ void __launch_bounds__(W, 1024 / W) verify_walk_kernel(const __grid_constant__ VerifyParams P) {
    extern __shared__ float kept[];                      // logits, then the draft's probabilities
    constexpr int RUN = ((VF_SLICE + W - 1) / W) | 1;
    __shared__ double node_z[VF_NODES], node_w[VF_NODES], part[W / 32], total_s[2], run_w[RUN];
    __shared__ float node_m[VF_NODES];
    __shared__ int node_at[VF_NODES], parent[VF_NODES], token[VF_NODES], next[VF_NODES], path[VF_NODES], gone[VF_NODES];
    __shared__ int length, n_gone, finder;
    pdl_wait();
    pdl_launch_dependents();
    const int b = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, n = nodes_of(P, b), T = P.T;
    const int rank = (int)cluster_rank(), ranks = (int)cluster_size();
    if (n == 0) {                                        // the whole cluster agrees
        if (rank == 0) {
            for (int i = tid; i < T; i += W) { P.path[(size_t)b * T + i] = -1; P.out[(size_t)b * T + i] = -1; }
            if (tid == 0) P.count[b] = -1;
        }
        return;
    }
    const float t = temperature_of(P, b);
    const bool greedy = !(t > 0.f);
    const double inv = greedy ? 1.0 : 1.0 / (double)t;
    if (tid < n) {
        const int p = P.parents ? P.parents[(size_t)b * T + tid] : tid - 1;
        parent[tid] = tid > 0 && p >= 0 && p < tid ? p : -1;             // a node without one is never reached
        token[tid] = P.tokens[(size_t)b * T + tid];
        next[tid] = VF_NODES;
    }
    if (tid == 0) { n_gone = 0; finder = W; }
    for (int i = warp; i < n; i += W / 32) {    // the chunks of a node's row
        const float4* st = P.stats + ((size_t)b * T + i) * P.chunks;
        float m = -INFINITY;
        int at = 0x7fffffff;
        for (int k = lane; k < P.chunks; k += 32) {
            const float4 c = st[k];
            const int ca = __float_as_int(c.z);
            if (c.x > m || (c.x == m && ca < at)) { m = c.x; at = ca; }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const float om = __shfl_xor_sync(0xffffffffu, m, o);
            const int oa = __shfl_xor_sync(0xffffffffu, at, o);
            if (om > m || (om == m && oa < at)) { m = om; at = oa; }
        }
        double z = 0;
        for (int k = lane; k < P.chunks; k += 32) {
            const float4 c = st[k];
            z += (double)c.y * weight(c.x, m, inv);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (lane == 0) { node_m[i] = m; node_at[i] = at; node_z[i] = z; }
    }
    __syncthreads();
    const bool child = tid < n && tid > 0 && parent[tid] >= 0;
    double wc = 0;
    if (child && !greedy && token[tid] >= 0 && token[tid] < P.V) {
        wc = weight(logit_at<BF16>(P, b, parent[tid], token[tid]), node_m[parent[tid]], inv);
        for (int j = 1; j < tid; ++j)
            if (parent[j] == parent[tid] && token[j] == token[tid]) wc = 0;       // nothing is left of a token that a sibling had
    }
    if (tid < n) node_w[tid] = wc;
    __syncthreads();
    if (child) {
        const int p = parent[tid];
        bool take;
        if (greedy) {
            take = token[tid] == node_at[p];
        } else {
            double left = node_z[p];
            for (int j = 1; j < tid; ++j)
                if (parent[j] == p) left -= node_w[j];
            if (P.probs) left *= token[tid] >= 0 && token[tid] < P.V ? (double)P.probs[(size_t)b * P.p_batch + (size_t)p * P.p_row + token[tid]] : 0.0;
            take = (double)P.u[(size_t)b * T + tid] * left < wc;
        }
        if (take) atomicMin(&next[p], tid);
    }
    __syncthreads();
    if (tid == 0) {
        int k = 0;
        path[0] = 0;
        while (next[path[k]] < VF_NODES) { path[k + 1] = next[path[k]]; ++k; }    // a child's number is above its parent's: it ends
        length = k;
    }
    __syncthreads();
    const int last = length, end = path[last];
    if (rank == 0) {
        for (int i = tid; i < T; i += W) {
            P.path[(size_t)b * T + i] = i <= last ? path[i] : -1;
            if (i != last) P.out[(size_t)b * T + i] = i < last ? token[path[i + 1]] : -1;
            else if (greedy) P.out[(size_t)b * T + i] = node_at[end];
        }
        if (tid == 0) P.count[b] = last;
    }
    if (greedy) return;
    if (child && parent[tid] == end) gone[atomicAdd(&n_gone, 1)] = token[tid];
    __syncthreads();
    const int v0 = rank * P.slice, len = max(0, min(P.slice, P.V - v0));
    const float m = node_m[end];
    for (int k = tid; k < len; k += W) kept[k] = logit_at<BF16>(P, b, end, v0 + k);
    const bool rest = P.probs && n_gone > 0;         // a child was rejected: what the draft's distribution leaves of the target's
    float* q = kept + P.slice;
    if (rest)
        for (int k = tid; k < len; k += W) q[k] = P.probs[(size_t)b * P.p_batch + (size_t)end * P.p_row + v0 + k];
    __syncthreads();
    if (!rest && tid < n_gone) {
        const int g = gone[tid] - v0;
        if (g >= 0 && g < len) kept[g] = -INFINITY;
    }
    __syncthreads();
    // each thread sums a run of neighbours (an odd number: no two lanes of a warp meet in a bank), the block scans the sums
    const int run = ((P.slice + W - 1) / W) | 1, k0 = min(len, tid * run), k1 = min(len, k0 + run);
    double z = 1.0;
    auto left = [&](int k) {                             // the weight of a token
        const double x = weight(kept[k], m, inv);
        return rest ? fmax(x / z - (double)q[k], 0.0) : x;
    };
    auto sum_run = [&] {
        double s = 0;
        for (int k = k0; k < k1; k += VF_TOGETHER) {     // several at a time: exponentials overlap
            double x[VF_TOGETHER];
#pragma unroll
            for (int i = 0; i < VF_TOGETHER; ++i) x[i] = k + i < k1 ? left(k + i) : 0.0;
#pragma unroll
            for (int i = 0; i < VF_TOGETHER; ++i) s += x[i];
        }
        return s;
    };
    if (rest) {                                          // first against nothing: the target's sum
        double s = 0;
        for (int k = k0; k < k1; ++k) s += weight(kept[k], m, inv);
        s = block_sum<W>(s, part);
        if (tid == 0) total_s[0] = s;
        cluster_sync();
        z = 0;
        for (int r = 0; r < ranks; ++r) z += ld_cluster_f64(smem_u32(&total_s[0]), r);
    }
    const double mine = sum_run();
    double upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += x;
    }
    if (lane == 31) part[warp] = upto;
    __syncthreads();
    if (warp == 0) {                                     // the warps' sums, scanned by one of them
        const double x = lane < W / 32 ? part[lane] : 0.0;
        double up = x;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double y = __shfl_up_sync(0xffffffffu, up, o);
            if (lane >= o) up += y;
        }
        if (lane < W / 32) part[lane] = up - x;
        if (lane == 31) total_s[1] = up;
    }
    __syncthreads();
    const double before = part[warp];
    cluster_sync();
    double sums[VF_CLUSTER], all = 0;
#pragma unroll
    for (int r = 0; r < VF_CLUSTER; ++r) sums[r] = r < ranks ? ld_cluster_f64(smem_u32(&total_s[1]), r) : 0.0;
#pragma unroll
    for (int r = 0; r < VF_CLUSTER; ++r) all += sums[r];
    const double target = (double)P.u[(size_t)b * T] * all;
    int owner = -1;
    double base = 0, run_sum = 0;
#pragma unroll
    for (int r = 0; r < VF_CLUSTER; ++r) {
        if (sums[r] > 0 && (owner < 0 || run_sum <= target)) { owner = r; base = run_sum; }       // the last part that starts at or below the target
        run_sum += sums[r];
    }
    cluster_sync();                                      // nobody leaves while its sums are read
    if (owner < 0) {                                     // nothing is left to draw from
        if (rank == 0 && tid == 0) P.out[(size_t)b * T + last] = node_at[end];
        return;
    }
    if (rank != owner) return;
    const double aim = target - base;
    if (mine > 0 && before + upto > aim) atomicMin(&finder, tid);
    __syncthreads();
    if (finder == W) {                          // rounding put the target behind the last sum: the last run with weight
        __syncthreads();
        if (tid == 0) finder = -1;
        __syncthreads();
        if (mine > 0) atomicMax(&finder, tid);
        __syncthreads();
    }
    const int found = finder, first = found * run, count = min(len, first + run) - first;      // the run that it falls into
    if (tid < count) run_w[tid] = left(first + tid);
    __syncthreads();
    if (tid == found) {
        double c = before + (upto - mine);
        int pick = -1;
        for (int k = 0; k < count; ++k) {
            if (run_w[k] <= 0) continue;
            pick = first + k;
            c += run_w[k];
            if (c > aim) break;
        }
        P.out[(size_t)b * T + last] = v0 + pick;
    }
}

template <bool BF16, int W>
int launch_walk(const VerifyParams& p, int cluster, cudaStream_t st) {
    static bool attr[64];
    int dev = 0;
    PTB_CUDA_OK(cudaGetDevice(&dev));
    if (dev >= 64 || !attr[dev]) {
        PTB_CUDA_OK(cudaFuncSetAttribute(verify_walk_kernel<BF16, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, VF_SLICE * 8));
        PTB_CUDA_OK(cudaFuncSetAttribute(verify_walk_kernel<BF16, W>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (dev < 64) attr[dev] = true;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(cluster, p.B);
    cfg.blockDim = dim3(W);
    cfg.dynamicSmemBytes = (size_t)p.slice * (p.probs ? 8 : 4);
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)cluster; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = ptb_pdl_enabled() ? 2 : 1;
    PTB_CUDA_OK(cudaLaunchKernelEx(&cfg, verify_walk_kernel<BF16, W>, p));
    return 0;
}

}  // namespace
}  // namespace ptb

using namespace ptb;

// Bytes of workspace that ptb_verify_drafts needs.
PTB_API long long ptb_verify_work_bytes(int B, int T, int V) { return (long long)B * T * ((V + VF_CHUNK - 1) / VF_CHUNK) * 16; }

// Which drafted tokens of B requests stay.  logits [B, T, V] (bf16 or fp32; pitches of a request and of a row in elements), tokens, parents (null: a chain) and u [B, T], nodes [B] (null: T),
// probs (null, or the draft's probabilities [B, T, V] fp32, row i what node i's child was drawn from; chains only), temperature [B].  Writes path [B, T] (accepted nodes, -1 behind),
// count [B] (accepted drafted tokens; -1 for a request without nodes) and out [B, T] (their tokens, then the drawn one, -1 behind).
PTB_API int ptb_verify_drafts(const void* logits, int bf16, long long l_batch, long long l_row, const float* probs, long long p_batch, long long p_row, const int* tokens, const int* parents,
                              const int* nodes, const float* u, const float* temperature, void* work, int* path, int* count, int* out, int B, int T, int V, cudaStream_t st) {
    if (B <= 0) return 0;
    if (T < 1 || T > VF_NODES || V < 1 || (long long)B * T > VF_ROWS || B > 65535 || V > VF_SLICE * VF_CLUSTER) {
        ptb_set_error("verify_drafts: %d requests of %d nodes over %d tokens (1 to %d nodes, %d in all, up to %d tokens)", B, T, V, VF_NODES, VF_ROWS, VF_SLICE * VF_CLUSTER);
        return -1;
    }
    if (probs && parents) { ptb_set_error("verify_drafts: draft probabilities go with chains"); return -1; }
    if (((uintptr_t)work & 15)) { ptb_set_error("verify_drafts: the workspace needs to be 16-byte aligned"); return -1; }
    VerifyParams p;
    p.logits = logits; p.l_batch = l_batch; p.l_row = l_row; p.probs = probs; p.p_batch = p_batch; p.p_row = p_row; p.tokens = tokens; p.parents = parents; p.nodes = nodes;
    p.u = u; p.temperature = temperature; p.stats = (float4*)work; p.path = path; p.count = count; p.out = out; p.B = B; p.T = T; p.V = V;
    p.chunks = (V + VF_CHUNK - 1) / VF_CHUNK;
    int cluster = 1;
    while (cluster < 8 && V > cluster * 2048) cluster *= 2;
    if (V > cluster * VF_SLICE) cluster = VF_CLUSTER;
    p.slice = (V + cluster - 1) / cluster;
    const int unit = bf16 ? 8 : 4;
    const bool vec = !((uintptr_t)logits & 15) && l_batch % unit == 0 && l_row % unit == 0;
    void (*k)(VerifyParams) = bf16 ? (vec ? verify_stats_kernel<true, true> : verify_stats_kernel<true, false>) : (vec ? verify_stats_kernel<false, true> : verify_stats_kernel<false, false>);
    PTB_CUDA_OK(ptb_launch(k, dim3(B * T * p.chunks), dim3(VF_THREADS), 0, st, ptb_pdl_enabled(), p));
    // threads of a CTA of the walk: 1024 where each finds an SM of its own, else two of 512 share one
    const bool wide = (long long)B * cluster <= VF_WIDE;
    if (bf16 ? (wide ? launch_walk<true, 1024>(p, cluster, st) : launch_walk<true, 512>(p, cluster, st)) : (wide ? launch_walk<false, 1024>(p, cluster, st) : launch_walk<false, 512>(p, cluster, st)))
        return -1;
    PTB_CUDA_OK(cudaGetLastError());
    return 0;
}
