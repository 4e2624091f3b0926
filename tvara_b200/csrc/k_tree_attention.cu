// Attention of drafted-token trees over the paged KV cache
// (tvara_tree_attention of include/tvara_kernels.h).
//
// Row i of sequence s, query head h:  o = sum_j w_j v_j,  w = softmax over
// the visible j of q.k_j / sqrt(d),  j running over the L cached positions
// (block table) and the nodes whose bit is set in the row's mask (slots).
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>

#include "tree.cuh"

namespace tvara {
namespace {

// The sequence of row t: the last one whose rows begin at or before it.
// False when the row belongs to none or its sequence's sizes are invalid.
__device__ __forceinline__ bool tree_sequence_ok(const TreeAttn& a, int s, int& c0, int& n, int& len) {
    c0 = a.cu[s];
    const int c1 = a.cu[s + 1];
    len = a.lengths[s];
    const long long rows = (long long)c1 - c0;
    n = int(rows);
    return c0 >= 0 && rows >= 0 && rows <= a.max_nodes && c1 <= a.capacity && len >= 0 &&
           len <= (long long)a.stride * a.bt;
}

// Element offset of the K row (head 0 of the layer) of index p of a sequence
// (cached positions, then nodes), or -1 with the status bit for a block or
// slot outside the pool.
__device__ __forceinline__ long long tree_row(const TreeAttn& a, int s, int c0, int len, int p, int& flags) {
    long long block, off;
    if (p < len) {
        const int e = p / a.bt;
        block = a.tables[(long long)s * a.stride + e];
        off = p - e * a.bt;
    } else {
        const long long slot = a.slots[c0 + p - len];
        block = slot < 0 ? -1 : slot / a.bt;
        off = slot - block * a.bt;
    }
    if (block < 0 || block >= a.max_blocks) {
        flags |= kTreeBadBlock;
        return -1;
    }
    return block * a.block_stride + a.layer_offset + off * a.dim;
}

// ---------------------------------------------------------- any shape
// One CTA of four warps per (row, query head), positions dealt to the warps,
// online softmax in F32, merged through shared memory.  Each position's K is
// reduced across the warp, so this form is bound by those shuffles (a few
// percent of memory bandwidth); it serves the shapes that the tensor-core
// form does not take (launch_tree_attention).
constexpr int kAnyWarps = 4;

__device__ __forceinline__ float kv_value(const TreeAttn& a, long long at) {
    if (a.kv_kind == 0) return static_cast<const float*>(a.kv)[at];
    if (a.kv_kind == 1) return __half2float(static_cast<const __half*>(a.kv)[at]);
    return float(static_cast<const signed char*>(a.kv)[at]);
}

template <int E>  // elements of a row per lane
__global__ void __launch_bounds__(kAnyWarps * 32) tree_any_kernel(TreeAttn a) {
    __shared__ float sm_m[kAnyWarps], sm_l[kAnyWarps];
    __shared__ float sm_acc[kAnyWarps][E * 32];
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (t >= a.cu[a.n_seq]) return;
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    int c0, n, len, flags = 0;
    const bool ok = tree_sequence_ok(a, lo, c0, n, len);
    if (!ok || t < c0 || t - c0 >= n) {
        if (threadIdx.x == 0 && h == 0) atomicOr(a.status, kTreeBadLengths);
        return;
    }
    const int node = t - c0, g = h / (a.hq / a.hkv);
    const unsigned long long* mask = a.ancestors ? a.ancestors + (long long)t * a.words : nullptr;
    const float* q = a.q + (long long)t * a.ldq + (long long)h * a.dim;
    float qv[E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = lane + 32 * e < a.dim ? q[lane + 32 * e] : 0.f;
        acc[e] = 0.f;
    }
    const float scale = 1.f / sqrtf(float(a.dim));
    float m = -INFINITY, l = 0.f;
    const long long end = (long long)len + n;
    for (long long p = warp; p < end; p += kAnyWarps) {
        if (p >= len) {
            const int j = int(p) - len;
            if (mask ? !((mask[j >> 6] >> (j & 63)) & 1) : j > node) continue;
        }
        const long long base = tree_row(a, lo, c0, len, int(p), flags);
        if (base < 0) continue;
        const long long k = base + (long long)g * a.bt * a.dim, v = k + a.kind_stride;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < a.dim) dot = fmaf(qv[e], kv_value(a, k + lane + 32 * e), dot);
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        float s = dot * scale, sv = 1.f;
        if (a.scales) {
            s *= a.scales[k / a.dim];
            sv = a.scales[v / a.dim];
        }
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float keep = expf(m - ref), w = expf(s - ref);
        m = mn;
        l = l * keep + w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < a.dim) acc[e] = fmaf(w * sv, kv_value(a, v + lane + 32 * e), acc[e] * keep);
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < kAnyWarps; ++w) top = fmaxf(top, sm_m[w]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int w = 0; w < kAnyWarps; ++w) total += sm_l[w] * expf(sm_m[w] - ref);
    for (int d = threadIdx.x; d < a.dim; d += kAnyWarps * 32) {
        float sum = 0.f;
        for (int w = 0; w < kAnyWarps; ++w) sum += sm_acc[w][d] * expf(sm_m[w] - ref);
        // NaN sums (non-finite inputs) stay NaN; a row that attends to nothing is zero
        a.out[(long long)t * a.ldo + (long long)h * a.dim + d] = total == 0.f && top == -INFINITY ? 0.f : sum / total;
    }
    if (flags && lane == 0) atomicOr(a.status, flags);
}

}  // namespace

std::size_t tree_attention_workspace(const TreeAttn&) { return 256; }

void launch_tree_attention(const TreeAttn& a, void*, cudaStream_t s) {
    const dim3 grid(unsigned(a.capacity), unsigned(a.hq));
    if (a.dim <= 32)
        tree_any_kernel<1><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (a.dim <= 64)
        tree_any_kernel<2><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (a.dim <= 128)
        tree_any_kernel<4><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else
        tree_any_kernel<8><<<grid, kAnyWarps * 32, 0, s>>>(a);
    TVARA_LAUNCHED();
}

}  // namespace tvara
